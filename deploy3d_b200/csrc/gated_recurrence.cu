// Gated linear recurrence over sequences of voxel rows, its backward pass, and its form for one row a sequence.
//   h[t] = f[t] h[t-1] + (1 - f[t]) x[t],  f = sigmoid(gate);  h in front of a sequence is initial[s] (zeros without)
//   delta[t] = grad[t] + f[t+1] delta[t+1]  (+ grad_final[s] at the last row),  dx = delta (1 - f),
//   dgate = delta (h[t-1] - x) f (1 - f),  dinitial[s] = f delta at the first row
// A row is the map c -> a c + b.  Maps compose: (a2, b2) after (a1, b1) is (a2 a1, a2 b1 + b2), so a tile of rows is one map per
// channel, and tiles can be worked on side by side: one kernel leaves the tiles' maps (and, for every sixteen rows, that of the
// tile's rows in front of them), one chains the tiles, one goes over the rows again, each sixteen on their own.  No thread of it
// waits for another CTA, and every sum is made in one order.  A row that starts a sequence is the map c -> b whatever c is, also
// where c is not finite: its a is -0, and the sign says that what came before is not looked at (products keep it, f is never
// negative).
// The rows are read twice, the second time in part from L2, and the gate is evaluated both times.  One kernel that hands the state
// from tile to tile would do either once; it has not been built, so what its waits would cost is not known.  Measured: 463 k x 64 bf16
// 73 us, maps 30, chain 8, rows 31 to 40 by what L2 still holds (178 MB of features in and out, floor 27 us); 120 k x 128 fp16 with
// gradients 109 us, maps 21 and 20, chains 5 and 5, rows 21 and 47.  Maps are bound by instructions (23 an element, 2.9 a cycle
// issued of 4), the rows by their bytes, backward by the 16 warps an SM that 128 registers leave.  Forward the last kernel
// spills 32 bytes a thread of paired 16-bit rows (64 registers, for four CTAs an SM).
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "packed.cuh"

namespace d3d {
namespace {

constexpr int kRows = 16;      // rows of a thread
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
  // between the kernels; a group are the kRows rows of a thread
  float2* prefix;   // [groups][channels] map of the tile's rows in front of the group, or behind it
  float2* maps;     // [tiles][channels] the tile's map
  float* carry;     // [tiles][channels] what comes into the tile
  uint4* marks;     // [groups] Marks
  float* states;    // [rows / kRows][channels] h in front of the group, from the forward pass to the backward pass
  int tiles;
};

__device__ __forceinline__ bool is_reset(float a) { return __float_as_int(a) < 0; }
__device__ __forceinline__ float reset_mark() { return __int_as_float((int)0x80000000u); }
// a h + b for the factor of several rows.  As a product of many gates it may have become zero although none of them is; walked row by
// row an infinite state stays one, so it does here: zero is taken as 2^-149 times 2^-149, which no number is left of.
__device__ __forceinline__ float carry_on(float a, float b, float h) {
  const float least = __int_as_float(1);
  return fmaf(a == 0.f ? least : a, h * (a == 0.f ? least : 1.f), b);
}
// The map (a, b) at h.
__device__ __forceinline__ float apply(float a, float b, float h) {
  const float r = carry_on(a, b, h);
  return is_reset(a) ? b : r;
}
// (a, b) after (pa, pb).
__device__ __forceinline__ void after(float& a, float& b, float pa, float pb) {
  b = apply(a, b, pb);
  a = is_reset(a) ? a : a * pa;
}

// f = sigmoid(gate) and 1 - f.  With t = exp(-|gate|) the smaller one is t / (1 + t), the other one a difference that loses
// nothing; with t = exp(-gate) the smaller one is t / (1 + t) while t < 1, then 1 / (1 + t), zero where t is infinite (463 k x 64 bf16
// 70.2 us; by exp(-|gate|) 76.8).
// Neither has a sign, NaN included: the sign of a map means a reset.
// Features of 32 bits: exponential and quotient to two units of the last place.  Of 16 bits: the hardware's base-two exponential,
// whose argument is rounded to |gate| 2^-24 (so that 1 - f is off by that much, relatively; the gate itself came rounded to 2^-9
// or 2^-12 of it), a third of the instructions.
template <class T, int V> __device__ __forceinline__ void gate_of(const Vec<V>& g, Vec<V>& f, Vec<V>& rest) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float t = expf(-fabsf(g.v[e])), small = t * __fdividef(1.f, 1.f + t), large = 1.f - small;
      f.v[e] = g.v[e] >= 0.f ? large : small, rest.v[e] = g.v[e] >= 0.f ? small : large;
    }
  } else {
    const Vec<V> y = mul(g, all<V>(-1.44269504f));
    Vec<V> t, r;
#pragma unroll
    for (int e = 0; e < V; ++e) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.v[e]) : "f"(y.v[e]));
    const Vec<V> d = add(t, all<V>(1.f));
#pragma unroll
    for (int e = 0; e < V; ++e) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.v[e]) : "f"(d.v[e]));
    const Vec<V> large = fma(r, all<V>(-1.f), all<V>(1.f));
#pragma unroll
    for (int e = 0; e < V; ++e) rest.v[e] = t.v[e] < 1.f ? t.v[e] * r.v[e] : large.v[e];
    f = fma(rest, all<V>(-1.f), all<V>(1.f));
#pragma unroll
    for (int e = 0; e < V; ++e) f.v[e] = t.v[e] < 1.f ? f.v[e] : r.v[e];
  }
}
// Both in one number: the smaller one, with a sign where that is f.
template <int V> __device__ __forceinline__ Vec<V> fold_gate(const Vec<V>& f, const Vec<V>& rest) {
  Vec<V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r.v[e] = f.v[e] < rest.v[e] ? -f.v[e] : rest.v[e];
  return r;
}
template <int V> __device__ __forceinline__ void open_gate(const Vec<V>& gate, Vec<V>& f, Vec<V>& rest) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const bool keeps = __float_as_int(gate.v[e]) >= 0;
    const float small = fabsf(gate.v[e]), large = 1.f - small;
    f.v[e] = keeps ? large : small, rest.v[e] = keeps ? small : large;
  }
}

// A thread's place: kLanes threads stand side by side along the channels, V channels each; the groups of them follow the rows,
// kRows each.  Tiles lie where they lie in the tensors, whatever the sequences cover, so that nothing has to be read before the
// rows are; walking down, they are counted from the end.
template <int V, int kLanes> struct Place {
  static constexpr int kWidth = V * kLanes, kGroups = kThreads / kLanes, kTile = kGroups * kRows;
  int tile, slab, lane, group, c, there;  // there: rows of the thread that the tensors have, a bit each
  int64_t low;                            // the tile's lowest row
  bool reverse;
  __device__ __forceinline__ explicit Place(const ScanArgs& a) {
    slab = blockIdx.x, tile = blockIdx.z * kTilesY + blockIdx.y, reverse = a.reverse != 0;
    lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, c = slab * kWidth + lane * V;
    low = (int64_t)(reverse ? a.tiles - 1 - tile : tile) * kTile;
    there = c < a.channels && tile < a.tiles ? (int)span(low_row(), 0, a.rows) : 0;
  }
  __device__ __forceinline__ int64_t low_row() const { return low + (reverse ? kTile - kRows - group * kRows : group * kRows); }
  // Of the sixteen rows from `from` on those in [begin, end), a bit each, in the order they are walked in.
  __device__ __forceinline__ uint32_t span(int64_t from, int64_t begin, int64_t end) const {
    const int64_t b = begin - from, e = end - from;
    const int lo = b < 0 ? 0 : b < kRows ? (int)b : kRows, hi = e < 0 ? 0 : e < kRows ? (int)e : kRows;
    const uint32_t up = hi > lo ? ((1u << hi) - 1) & ~((1u << lo) - 1) : 0u;
    return reverse ? __brev(up) >> (32 - kRows) : up;
  }
  // The thread's first row walked and its address in rows `ld` elements apart, with the distance to the next one.
  __device__ __forceinline__ int64_t first_row() const { return low_row() + (reverse ? kRows - 1 : 0); }
  template <class T> __device__ __forceinline__ T* start(T* base, int64_t ld) const { return base + first_row() * ld + c; }
  __device__ __forceinline__ int64_t step(int64_t ld) const { return reverse ? -ld : ld; }
  __device__ __forceinline__ int64_t group_id() const { return (int64_t)tile * kGroups + group; }
  __device__ __forceinline__ int64_t state_row() const { return low_row() / kRows; }  // the same for tiles of any shape
};

// kPastL1: from L2, for the last kernels, which read their rows before they wait for the ones in front of them (463 k x 64 bf16 73.5 us,
// waiting first 76.4).  What wrote the rows has ended by then, since the first kernel lets the others start when it has waited for
// it, but L1 need not know.
template <class T, int V, bool kPastL1> __device__ __forceinline__ Pack<T, V> load_row(const T* p) {
  if constexpr (!kPastL1) return *reinterpret_cast<const Pack<T, V>*>(p);
  Pack<T, V> r;
  static_assert(sizeof(r) == 4 || sizeof(r) == 2, "one or two channels");
  if constexpr (sizeof(r) == 4) {
    const uint32_t bits = __ldcg(reinterpret_cast<const uint32_t*>(p));
    memcpy(&r, &bits, 4);
  } else {
    const uint16_t bits = __ldcg(reinterpret_cast<const unsigned short*>(p));
    memcpy(&r, &bits, 2);
  }
  return r;
}

template <class T, int V, int kLanes, bool kPastL1 = false>
__device__ __forceinline__ void load_rows(Pack<T, V> (&to)[kRows], const Place<V, kLanes>& at, const void* p, int64_t ld) {
  const T* src = at.start((const T*)p, ld);
  const int64_t step = at.step(ld);
  if (at.there == (1 << kRows) - 1) {
#pragma unroll
    for (int r = 0; r < kRows; ++r, src += step) to[r] = load_row<T, V, kPastL1>(src);
  } else {
    asm("" : "+l"(src));  // the addresses are those above, but need not all be there before the branch
#pragma unroll
    for (int r = 0; r < kRows; ++r, src += step)
      if (at.there >> r & 1) to[r] = load_row<T, V, kPastL1>(src);
  }
}
template <int V> __device__ __forceinline__ Vec<V> load_state(const float* p, int64_t s, int channels, int c) {
  Vec<V> r = all<V>(0.f);
  if (p)
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = load_fresh(p + s * channels + c + e);
  return r;
}
template <int V> __device__ __forceinline__ void store_state(float* p, int64_t s, int channels, int c, const Vec<V>& h) {
  if (p)
#pragma unroll
    for (int e = 0; e < V; ++e) p[s * channels + c + e] = h.v[e];
}

// The last sequence that starts at or before row t, by a whole warp: 32 probes a step.
__device__ __forceinline__ int sequence_of(const ScanArgs& a, int64_t t) {
  int lo = 0, n = a.seqs;
  while (n > 1) {
    const int step = (n + 31) / 32, at = lo + lane_id() * step;
    const unsigned before = __ballot_sync(0xffffffffu, at < lo + n && load_fresh(a.offsets + at) <= t);
    const int k = before ? __popc(before) - 1 : 0, end = lo + n;
    lo += k * step;
    if (lo > end - 1) lo = end - 1;  // offsets out of order
    n = end - lo < step ? end - lo : step;
  }
  return lo;
}
// Of the marked rows of a thread, one after the other in the order they are walked in: whose they are.  s: the sequence of the
// lowest row around.
struct Finder {
  int s;
  __device__ __forceinline__ int of(const ScanArgs& a, int64_t t) {
    while (s + 1 < a.seqs && load_fresh(a.offsets + s + 1) <= t) ++s;
    while (s > 0 && load_fresh(a.offsets + s) > t) --s;
    return s;
  }
};

// Which rows of a thread sequences have, and where they start and end, in the order they are walked in: a bit per row.
struct Marks {
  uint32_t live;  // those of the tensors that a sequence has
  uint32_t ends;  // starts in the low half, ends in the high one
  int owner;      // sequence of the lowest row of the warp
  __device__ __forceinline__ bool plain(uint32_t which) const { return live == (1u << kRows) - 1 && (ends & which) == 0; }
};
// By every warp for its own rows, which follow one another: the sequences from that of the lowest row on, a lane each.
template <int V, int kLanes>
__device__ __forceinline__ Marks mark_ends(const ScanArgs& a, const Place<V, kLanes>& at) {
  constexpr int kSpan = kRows * (32 / kLanes), kTile = Place<V, kLanes>::kTile;  // rows of a warp: 16, 32 or 64
  const int front = (int)(threadIdx.x >> 5) * kSpan;
  const int64_t low = at.low + (at.reverse ? kTile - front - kSpan : front);
  const int owner = sequence_of(a, low);
  uint32_t first[kSpan > 32 ? 2 : 1] = {}, last[kSpan > 32 ? 2 : 1] = {};
  for (int base = owner; base < a.seqs; base += 32) {
    const int s = base + lane_id();
    const bool in = s < a.seqs;
    const int64_t b = in ? (int64_t)load_fresh(a.offsets + s) - low : kSpan, e = in ? (int64_t)load_fresh(a.offsets + s + 1) - 1 - low : kSpan;
    if (b <= e) {
      if (b >= 0 && b < kSpan) first[kSpan > 32 ? (int)b >> 5 : 0] |= 1u << ((int)b & 31);
      if (e >= 0 && e < kSpan) last[kSpan > 32 ? (int)e >> 5 : 0] |= 1u << ((int)e & 31);
    }
    if (__any_sync(0xffffffffu, b >= kSpan)) break;  // past the highest row
  }
  // of the warp's rows, upwards, to the thread's sixteen, as they are walked
  uint64_t f = 0, l = 0;
#pragma unroll
  for (int w = 0; w < (kSpan > 32 ? 2 : 1); ++w) {
    f |= (uint64_t)__reduce_or_sync(0xffffffffu, first[w]) << (32 * w);
    l |= (uint64_t)__reduce_or_sync(0xffffffffu, last[w]) << (32 * w);
  }
  if (at.reverse) {
    const uint64_t up = f;  // walking down starts where a sequence ends
    f = __brevll(l) >> (64 - kSpan), l = __brevll(up) >> (64 - kSpan);
  }
  const int shift = lane_id() / kLanes * kRows;
  const uint32_t live = at.there & at.span(at.low_row(), load_fresh(a.offsets), load_fresh(a.offsets + a.seqs));
  const uint32_t starts = (uint32_t)(f >> shift) & live, ends = (uint32_t)(l >> shift) & live;
  return {live, starts | ends << 16, owner};
}

// From the maps of the threads' rows to that of the tile and, for every thread, that of the rows of the tile in front of its own
// (kUp) or behind them; both go to memory, with the marks.  The channels' chains over the warps are walked by a thread each.
template <int V, int kLanes, bool kUp> struct Chain {
  static constexpr int kWidth = V * kLanes, kGroups = kThreads / kLanes;
  float2 totals[kWarps][kWidth];

  // Every thread brings its map; behind a barrier the warps' lie in `totals`.
  __device__ __forceinline__ void bring(Vec<V>& ma, Vec<V>& mb, const Place<V, kLanes>& at) {
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
      for (int e = 0; e < V; ++e) totals[warp][col + e] = make_float2(ma.v[e], mb.v[e]);
  }
  // The chain of a channel: to(warp, map of the warps on the way to it) for each; the map of all.
  template <class F> __device__ __forceinline__ float2 walk(int t, F to) {
    float pa = 1.f, pb = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const int w = kUp ? i : kWarps - 1 - i;
      float2 m = totals[w][t];
      to(w, make_float2(pa, pb));
      after(m.x, m.y, pa, pb);
      pa = m.x, pb = m.y;
    }
    return make_float2(pa, pb);
  }
  // Behind a chain that has left its maps in `totals`: that of the rows on the way to the thread's, of its channel `e`.
  __device__ __forceinline__ float2 own(const Vec<V>& ma, const Vec<V>& mb, const Place<V, kLanes>& at, int e) const {
    const int lane = lane_id();
    const float2 front = totals[threadIdx.x >> 5][at.lane * V + e];
    if constexpr (kLanes < 32) {  // several groups in a warp
      float pa = kUp ? __shfl_up_sync(0xffffffffu, ma.v[e], kLanes) : __shfl_down_sync(0xffffffffu, ma.v[e], kLanes);
      float pb = kUp ? __shfl_up_sync(0xffffffffu, mb.v[e], kLanes) : __shfl_down_sync(0xffffffffu, mb.v[e], kLanes);
      if (kUp ? lane >= kLanes : lane + kLanes < 32) {
        after(pa, pb, front.x, front.y);
        return make_float2(pa, pb);
      }
    }
    return front;
  }

  __device__ __forceinline__ void finish(const ScanArgs& a, Vec<V> ma, Vec<V> mb, const Place<V, kLanes>& at, const Marks& marks) {
    bring(ma, mb, at);
    if (at.slab == 0 && at.lane == 0) a.marks[at.group_id()] = make_uint4(marks.live, marks.ends, (uint32_t)marks.owner, 0u);
    __syncthreads();
    const int t = threadIdx.x, c = at.slab * kWidth + t;
    if (t < kWidth && c < a.channels) {
      float2* to = a.prefix + (int64_t)at.tile * kGroups * a.channels + c;
      a.maps[(int64_t)at.tile * a.channels + c] = walk(t, [&](int w, float2 m) {
        if constexpr (kLanes == 32) to[w * a.channels] = m;
        else totals[w][t] = m;
      });
    }
    if constexpr (kLanes < 32) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 m = own(ma, mb, at, e);
        if (at.c < a.channels) a.prefix[at.group_id() * a.channels + at.c + e] = m;
      }
    }
  }
  // The same for the only tile, into which nothing comes: what comes into the thread's rows.
  __device__ __forceinline__ Vec<V> only(Vec<V> ma, Vec<V> mb, const Place<V, kLanes>& at) {
    bring(ma, mb, at);
    __syncthreads();
    if (threadIdx.x < kWidth) walk(threadIdx.x, [&](int w, float2 m) { totals[w][threadIdx.x] = m; });
    __syncthreads();
    Vec<V> h;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float2 m = own(ma, mb, at, e);
      h.v[e] = apply(m.x, m.y, 0.f);
    }
    return h;
  }
};

// What comes into the thread's rows: the tile's rows on the way, after what comes into the tile.
template <int V, int kLanes>
__device__ __forceinline__ Vec<V> incoming(const ScanArgs& a, const Place<V, kLanes>& at) {
  Vec<V> h = all<V>(0.f);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float2 m = __ldcg(a.prefix + at.group_id() * a.channels + at.c + e);
    h.v[e] = apply(m.x, m.y, __ldcg(a.carry + (int64_t)at.tile * a.channels + at.c + e));
  }
  return h;
}

// Sequences without rows: their last state is the one they start with.
template <int V, int kLanes>
__device__ __forceinline__ void pass_empty(const ScanArgs& a, const Place<V, kLanes>& at, const float* from, float* to) {
  if (!to) return;
  const int tiles = a.tiles > 0 ? a.tiles : 1, low = at.slab * V * kLanes;
  const int high = low + V * kLanes < a.channels ? low + V * kLanes : a.channels;
  for (int64_t s = (int64_t)at.tile * kThreads + threadIdx.x; s < a.seqs; s += (int64_t)tiles * kThreads)
    if (load_fresh(a.offsets + s + 1) <= load_fresh(a.offsets + s))
      for (int c = low; c < high; ++c) to[s * a.channels + c] = from ? load_fresh(from + s * a.channels + c) : 0.f;
}

// The map of a thread's rows, those from the last start of a sequence on: what was in front of it is gone.  Rows between two ends of
// sequences, all but a few, take a path without the tests, here and below.
template <class T, int V, int kLanes>
__device__ __forceinline__ void map_rows(const ScanArgs& a, const Place<V, kLanes>& at, const Marks& marks, const Pack<T, V> (&x)[kRows],
                                         const Pack<T, V> (&g)[kRows], Vec<V>& ma, Vec<V>& mb) {
  ma = all<V>(1.f), mb = all<V>(0.f);
  auto enter = [&](auto is_plain) {
    constexpr bool kPlain = decltype(is_plain)::value;
    Finder find = {marks.owner};
    const int64_t t = at.first_row(), step = at.step(1);
    const int from = 31 - __clz((int)(marks.ends & 0xffffu));
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (kPlain || (r >= from && (marks.live >> r & 1))) {
        Vec<V> f, rest;
        gate_of<T, V>(widen<T, V>(g[r]), f, rest);
        const Vec<V> u = mul(rest, widen<T, V>(x[r]));
        if (!kPlain && r == from) {
          mb = fma(f, load_state<V>(a.initial, find.of(a, t + r * step), a.channels, at.c), u);
          ma = all<V>(reset_mark());
        } else {
          mb = fma(f, mb, u), ma = mul(ma, f);
        }
      }
  };
  if (marks.plain(0xffffu)) enter(std::true_type());
  else enter(std::false_type());
}

// First kernel: maps.
template <class T, int V, int kLanes>
__global__ void __launch_bounds__(kThreads, 4)
scan_maps_kernel(const ScanArgs a) {
  __shared__ Chain<V, kLanes, true> chain;
  const Place<V, kLanes> at(a);
  if (at.tile >= a.tiles) return;  // the last thousands of tiles are not all there
  pdl_wait();
  pdl_release();  // behind the wait: the last kernel reads its rows before it waits, relying on this one
  Pack<T, V> x[kRows], g[kRows];
  load_rows<T, V, kLanes>(x, at, a.x, a.x_ld);
  load_rows<T, V, kLanes>(g, at, a.gates, a.gates_ld);
  const Marks marks = mark_ends(a, at);
  Vec<V> ma, mb;
  map_rows<T, V, kLanes>(a, at, marks, x, g, ma, mb);
  chain.finish(a, ma, mb, at, marks);
}

// What comes into each tile: the tiles' maps one after the other, from the first (or, backwards, the last) on.  Two channels to a
// CTA; 256 threads of each take kHeld tiles into registers, chain them, and are chained by shuffles and through shared memory.
constexpr int kHeld = 16, kCarryThreads = 512, kCarryChannels = 2, kCarryWarps = kCarryThreads / 32;
__global__ void __launch_bounds__(kCarryThreads)
carry_kernel(const float2* maps, float* __restrict__ into, int tiles, int channels, int backward) {
  __shared__ float2 totals[kCarryWarps][kCarryChannels];
  __shared__ float starts[kCarryWarps][kCarryChannels];
  const int lane = lane_id(), warp = threadIdx.x >> 5, ch = threadIdx.x % kCarryChannels, c = blockIdx.x * kCarryChannels + ch;
  const int segment = threadIdx.x / kCarryChannels;
  pdl_release();
  pdl_wait();
  float carry = 0.f;  // of channel `warp` of this CTA, in the warps that chain
  constexpr int kTurn = kCarryThreads / kCarryChannels * kHeld;
  float2 next[kHeld];
  auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int t = t0 + segment * kHeld + i;
      next[i] = make_float2(1.f, 0.f);
      if (t < tiles && c < channels) next[i] = __ldcg(maps + (int64_t)(backward ? tiles - 1 - t : t) * channels + c);
    }
  };
  load(0);
  for (int t0 = 0; t0 < tiles; t0 += kTurn) {
    float2 m[kHeld];
    float a = 1.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) m[i] = next[i];
    if (t0 + kTurn < tiles) load(t0 + kTurn);
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
      float2 w = lane < kCarryWarps ? totals[lane][warp] : make_float2(1.f, 0.f);
#pragma unroll
      for (int d = 1; d < kCarryWarps; d <<= 1) {
        const float pa = __shfl_up_sync(0xffffffffu, w.x, d), pb = __shfl_up_sync(0xffffffffu, w.y, d);
        if (lane >= d) after(w.x, w.y, pa, pb);
      }
      const float end = apply(w.x, w.y, carry), before = __shfl_up_sync(0xffffffffu, end, 1);
      if (lane < kCarryWarps) starts[lane][warp] = lane ? before : carry;
      carry = __shfl_sync(0xffffffffu, end, kCarryWarps - 1);
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

// Where sequences are short, their states are fetched for as many rows at once.
constexpr int kAhead = 4;

// Last kernel: the rows, each thread its own from what comes into them.  No thread waits for another.  kOnly: there is one
// tile, and this kernel does the others' work as well.
template <class T, int V, int kLanes, bool kOnly>
__global__ void __launch_bounds__(kThreads, 4)
scan_rows_kernel(const ScanArgs a) {
  const Place<V, kLanes> at(a);
  if (kOnly) pdl_wait();
  Pack<T, V> x[kRows], g[kRows];
  load_rows<T, V, kLanes, !kOnly>(x, at, a.x, a.x_ld);
  load_rows<T, V, kLanes, !kOnly>(g, at, a.gates, a.gates_ld);
  if (!kOnly) pdl_wait();
  Marks marks = {0u, 0u, 0};
  Vec<V> h;
  if constexpr (kOnly) {
    __shared__ Chain<V, kLanes, true> chain;
    Vec<V> ma, mb;
    marks = mark_ends(a, at);
    map_rows<T, V, kLanes>(a, at, marks, x, g, ma, mb);
    h = chain.only(ma, mb, at);
  } else if (at.there) {
    const uint4 word = __ldcg(a.marks + at.group_id());
    marks = {word.x & (uint32_t)at.there, word.y, (int)word.z};
    h = incoming<V, kLanes>(a, at);
  }
  if (at.there) {
    store_state<V>(a.states, at.state_row(), a.channels, at.c, h);
    T* out = at.start((T*)a.out, a.channels);
    const int64_t step = at.step(a.channels);
    auto walk = [&](auto is_plain) {
      constexpr bool kPlain = decltype(is_plain)::value;
      Finder find = {marks.owner}, from = find;
      const int64_t t = at.first_row(), next = at.step(1);
      Vec<V> start[kAhead];
#pragma unroll
      for (int r = 0; r < kRows; ++r, out += step) {
        if (!kPlain && r % kAhead == 0)
#pragma unroll
          for (int i = r; i < r + kAhead; ++i)
            if (marks.ends >> i & 1) start[i - r] = load_state<V>(a.initial, from.of(a, t + i * next), a.channels, at.c);
        if (kPlain || (marks.live >> r & 1)) {
          if (!kPlain && (marks.ends >> r & 1)) h = start[r % kAhead];
          Vec<V> f, rest;
          gate_of<T, V>(widen<T, V>(g[r]), f, rest);
          h = fma(f, h, mul(rest, widen<T, V>(x[r])));
          *reinterpret_cast<Pack<T, V>*>(out) = narrow<T, V>(h);
          if (!kPlain && (marks.ends >> (r + 16) & 1)) store_state<V>(a.final_state, find.of(a, t + r * next), a.channels, at.c, h);
        }
      }
    };
    if (marks.plain(~0u)) walk(std::true_type());
    else walk(std::false_type());
  }
  pass_empty<V, kLanes>(a, at, a.initial, a.final_state);
}

// Backward: gradients are carried from the end.  The map of a row is c -> f (grad + c): c comes in from the row behind and goes out
// to the row in front.
template <class T, int V, int kLanes>
__device__ __forceinline__ void map_rows_back(const ScanArgs& a, const Place<V, kLanes>& at, const Marks& marks, const Pack<T, V> (&g)[kRows],
                                              const Pack<T, V> (&d)[kRows], Vec<V>& ma, Vec<V>& mb) {
  ma = all<V>(1.f), mb = all<V>(0.f);
  auto enter = [&](auto is_plain) {
    constexpr bool kPlain = decltype(is_plain)::value;
    Finder find = {marks.owner};
    const int64_t t = at.first_row(), step = at.step(1);
    const int from = (marks.ends >> 16) ? __ffs((int)(marks.ends >> 16)) - 1 : kRows;
#pragma unroll
    for (int r = kRows - 1; r >= 0; --r)
      if (kPlain || (r <= from && (marks.live >> r & 1))) {
        Vec<V> f, rest;
        gate_of<T, V>(widen<T, V>(g[r]), f, rest);
        const Vec<V> dy = widen<T, V>(d[r]);
        if (!kPlain && r == from) {
          mb = mul(f, add(dy, load_state<V>(a.grad_final, find.of(a, t + r * step), a.channels, at.c)));
          ma = all<V>(reset_mark());
        } else {
          mb = mul(f, add(dy, mb)), ma = mul(ma, f);
        }
      }
  };
  if (marks.plain(0xffff0000u)) enter(std::true_type());
  else enter(std::false_type());
}

template <class T, int V, int kLanes>
__global__ void __launch_bounds__(kThreads, 4)
scan_backward_maps_kernel(const ScanArgs a) {
  __shared__ Chain<V, kLanes, false> chain;
  const Place<V, kLanes> at(a);
  if (at.tile >= a.tiles) return;
  pdl_wait();
  pdl_release();
  Pack<T, V> g[kRows], d[kRows];
  load_rows<T, V, kLanes>(g, at, a.gates, a.gates_ld);
  load_rows<T, V, kLanes>(d, at, a.grad, a.grad_ld);
  const Marks marks = mark_ends(a, at);
  Vec<V> ma, mb;
  map_rows_back<T, V, kLanes>(a, at, marks, g, d, ma, mb);
  chain.finish(a, ma, mb, at, marks);
}

// The rows forward once more from the state in front of them, which gives h[t-1] - x, then back with the gradients.
template <class T, int V, int kLanes, bool kOnly>
__global__ void __launch_bounds__(kThreads, 2)
scan_backward_rows_kernel(const ScanArgs a) {
  const Place<V, kLanes> at(a);
  if (kOnly) pdl_wait();
  Pack<T, V> x[kRows], g[kRows], d[kRows];
  load_rows<T, V, kLanes, !kOnly>(x, at, a.x, a.x_ld);
  load_rows<T, V, kLanes, !kOnly>(g, at, a.gates, a.gates_ld);
  load_rows<T, V, kLanes, !kOnly>(d, at, a.grad, a.grad_ld);
  if (!kOnly) pdl_wait();
  Marks marks = {0u, 0u, 0};
  Vec<V> q, h = all<V>(0.f);
  if constexpr (kOnly) {
    __shared__ Chain<V, kLanes, false> chain;
    Vec<V> ma, mb;
    marks = mark_ends(a, at);
    map_rows_back<T, V, kLanes>(a, at, marks, g, d, ma, mb);
    q = chain.only(ma, mb, at);
  } else if (at.there) {
    const uint4 word = __ldcg(a.marks + at.group_id());
    marks = {word.x & (uint32_t)at.there, word.y, (int)word.z};
    q = incoming<V, kLanes>(a, at);
  }
  if (at.there) {
    h = load_state<V>(a.states, at.state_row(), a.channels, at.c);
    const int64_t step = at.step(a.channels);
    T* dx_at = at.start((T*)a.grad_x, a.channels) + (kRows - 1) * step;
    T* dg_at = at.start((T*)a.grad_gates, a.channels) + (kRows - 1) * step;
    auto walk = [&](auto is_plain) {
      constexpr bool kPlain = decltype(is_plain)::value;
      Finder find = {marks.owner};
      const int64_t t = at.first_row(), next = at.step(1);
      Vec<V> gate[kRows], away[kRows], start[kAhead];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (!kPlain && r % kAhead == 0)
#pragma unroll
          for (int i = r; i < r + kAhead; ++i)
            if (marks.ends >> i & 1) start[i - r] = load_state<V>(a.initial, find.of(a, t + i * next), a.channels, at.c);
        if (kPlain || (marks.live >> r & 1)) {
          Vec<V> f, rest;
          gate_of<T, V>(widen<T, V>(g[r]), f, rest);
          gate[r] = fold_gate<V>(f, rest);
          if (!kPlain && (marks.ends >> r & 1)) h = start[r % kAhead];
          const Vec<V> in = widen<T, V>(x[r]);
          away[r] = fma(in, all<V>(-1.f), h);
          h = fma(f, h, mul(rest, in));
        }
      }
      Finder from = find;
#pragma unroll
      for (int r = kRows - 1; r >= 0; --r, dx_at -= step, dg_at -= step) {
        if (!kPlain && r % kAhead == kAhead - 1)
#pragma unroll
          for (int i = r; i > r - kAhead; --i)
            if (marks.ends >> (i + 16) & 1) start[i % kAhead] = load_state<V>(a.grad_final, from.of(a, t + i * next), a.channels, at.c);
        if (kPlain || (marks.live >> r & 1)) {
          Vec<V> f, rest;
          open_gate<V>(gate[r], f, rest);
          if (!kPlain && (marks.ends >> (r + 16) & 1)) q = start[r % kAhead];
          const Vec<V> delta = add(widen<T, V>(d[r]), q), dx = mul(delta, rest);
          q = mul(f, delta);
          *reinterpret_cast<Pack<T, V>*>(dx_at) = narrow<T, V>(dx);
          *reinterpret_cast<Pack<T, V>*>(dg_at) = narrow<T, V>(mul(mul(q, rest), away[r]));
          if (!kPlain && (marks.ends >> r & 1)) store_state<V>(a.grad_initial, find.of(a, t + r * next), a.channels, at.c, q);
        }
      }
    };
    if (marks.plain(~0u)) walk(std::true_type());
    else walk(std::false_type());
  }
  pass_empty<V, kLanes>(a, at, a.grad_final, a.grad_initial);
}

// One row a sequence: the state is read, moved on and written; state_out may be state.
template <class T, int V>
__global__ void __launch_bounds__(256)
step_kernel(const T* x, int64_t x_ld, const T* gates, int64_t gates_ld, const float* state,
            float* state_out, T* out, int64_t rows, int channels) {
  using P = Pack<T, V>;
  pdl_wait();
  pdl_release();
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

// f(V, lanes) for the tile shape: of 16-bit features two channels a thread where rows can be read so, else one, and as few threads
// side by side as cover the channels.
template <class T, class F> int by_shape(bool pairs, int channels, F f) {
#define D3D_SCAN_SHAPE(V, L) return f(std::integral_constant<int, V>(), std::integral_constant<int, L>())
  if constexpr (sizeof(T) == 2) {
    if (pairs) {
      if (channels <= 16) D3D_SCAN_SHAPE(2, 8);
      if (channels <= 32) D3D_SCAN_SHAPE(2, 16);
      D3D_SCAN_SHAPE(2, 32);
    }
  }
  if (channels <= 8) D3D_SCAN_SHAPE(1, 8);
  if (channels <= 16) D3D_SCAN_SHAPE(1, 16);
  D3D_SCAN_SHAPE(1, 32);
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
  D3D_REQUIRE(a.rows < (1ll << 31) && a.channels <= (1 << 16), D3D_ERR_TOO_LARGE);
  D3D_REQUIRE(on_multiples(dtype_size(dtype), a.x, a.gates, a.out, a.grad, a.grad_x, a.grad_gates) &&
                  on_multiples(4, a.offsets, a.initial, a.final_state, a.states, a.grad_final, a.grad_initial),
              D3D_ERR_INVALID_ARGUMENT);
  return D3D_OK;
}

// Between the kernels, sized for the smallest tiles and for whole ones of any shape.
constexpr int kSmallTile = kWarps * kRows, kMostGroups = kThreads / 8;
void carve(ScanArgs& a, Carver& w) {
  const size_t groups = (size_t)ceil_div(a.rows, kRows) + kMostGroups, tiles = (size_t)ceil_div(a.rows, kSmallTile) + 1;
  a.prefix = w.take<float2>(groups * a.channels);
  a.maps = w.take<float2>(tiles * a.channels);
  a.carry = w.take<float>(tiles * a.channels);
  a.marks = w.take<uint4>(groups);
}

// The three kernels of a pass, or for one tile the last one alone: two launches less where launches are what such a call lasts.
template <class Maps, class Rows>
int launch_pass(ScanArgs a, int tile, int width, Maps maps, Rows rows, Rows only, int backward, cudaStream_t st) {
  a.tiles = (int)ceil_div(a.rows, tile);
  const dim3 grid = grid_of(a.tiles, ceil_div(a.channels, width));
  if (a.tiles <= 1) {
    D3D_LAUNCH(true, only, grid, kThreads, 0, st, a);
    return D3D_OK;
  }
  D3D_LAUNCH(true, maps, grid, kThreads, 0, st, a);
  D3D_LAUNCH(true, carry_kernel, (unsigned)ceil_div(a.channels, kCarryChannels), kCarryThreads, 0, st, a.maps, a.carry, a.tiles,
             a.channels, backward);
  D3D_LAUNCH(true, rows, grid, kThreads, 0, st, a);
  return D3D_OK;
}

}  // namespace
}  // namespace d3d

using namespace d3d;

extern "C" int64_t d3d_gated_recurrence_state_rows(int64_t rows) { return rows < 0 ? 0 : ceil_div(rows > 0 ? rows : 1, kRows); }

extern "C" size_t d3d_gated_recurrence_workspace(int64_t rows, int channels) {
  if (rows <= kSmallTile || channels < 1) return 0;  // one tile of any shape
  ScanArgs a = {};
  a.rows = rows, a.channels = channels;
  Carver w(nullptr);
  carve(a, w);
  return w.off;
}

extern "C" int d3d_gated_recurrence(int dtype, const void* x, int64_t x_ld, const void* gates, int64_t gates_ld,
                                    const int32_t* offsets, int seqs, int64_t rows, int channels, int reverse,
                                    const float* initial, void* out, float* final_state, float* states, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  D3D_NVTX_RANGE("d3d_gated_recurrence");
  ScanArgs a = {};
  a.x = x, a.x_ld = x_ld, a.gates = gates, a.gates_ld = gates_ld, a.offsets = offsets, a.seqs = seqs, a.rows = rows;
  a.channels = channels, a.reverse = reverse != 0, a.initial = initial, a.out = out, a.final_state = final_state, a.states = states;
  const int rc = check_scan(dtype, a);
  D3D_REQUIRE(rc == D3D_OK, rc);
  D3D_REQUIRE(rows == 0 || (x && gates && out), D3D_ERR_INVALID_ARGUMENT);
  const size_t need = d3d_gated_recurrence_workspace(rows, channels);
  D3D_REQUIRE(need == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 256 == 0), D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace_bytes >= need, D3D_ERR_WORKSPACE_TOO_SMALL);
  Carver w(workspace);
  carve(a, w);
  if (seqs == 0) return D3D_OK;
  const int esize = (int)dtype_size(dtype);
  const bool pairs = channels % 2 == 0 && rows_paired(x, x_ld, esize) && rows_paired(gates, gates_ld, esize) && rows_paired(out, channels, esize);
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return by_shape<T>(pairs, channels, [&](auto v, auto l) -> int {
      constexpr int V = decltype(v)::value, L = decltype(l)::value;
      return launch_pass(a, Place<V, L>::kTile, V * L, scan_maps_kernel<T, V, L>, scan_rows_kernel<T, V, L, false>,
                         scan_rows_kernel<T, V, L, true>, 0,
                         reinterpret_cast<cudaStream_t>(stream));
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
  a.states = const_cast<float*>(states);
  const int rc = check_scan(dtype, a);
  D3D_REQUIRE(rc == D3D_OK, rc);
  D3D_REQUIRE(grad_ld >= channels && (rows == 0 || (x && gates && grad && states && grad_x && grad_gates)),
              D3D_ERR_INVALID_ARGUMENT);
  const size_t need = d3d_gated_recurrence_workspace(rows, channels);
  D3D_REQUIRE(need == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 256 == 0), D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace_bytes >= need, D3D_ERR_WORKSPACE_TOO_SMALL);
  Carver w(workspace);
  carve(a, w);
  if (seqs == 0) return D3D_OK;
  const int esize = (int)dtype_size(dtype);
  const bool pairs = channels % 2 == 0 && rows_paired(x, x_ld, esize) && rows_paired(gates, gates_ld, esize) &&
                     rows_paired(grad, grad_ld, esize) && rows_paired(grad_x, channels, esize) && rows_paired(grad_gates, channels, esize);
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return by_shape<T>(pairs, channels, [&](auto v, auto l) -> int {
      constexpr int V = decltype(v)::value, L = decltype(l)::value;
      return launch_pass(a, Place<V, L>::kTile, V * L, scan_backward_maps_kernel<T, V, L>,
                         scan_backward_rows_kernel<T, V, L, false>, scan_backward_rows_kernel<T, V, L, true>, 1,
                         reinterpret_cast<cudaStream_t>(stream));
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
  D3D_REQUIRE(x && gates && state && state_out && out && on_multiples(esize, x, gates, out) && on_multiples(4, state, state_out),
              D3D_ERR_INVALID_ARGUMENT);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto wide_rows = [esize](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * esize % 16 == 0; };
  const bool wide = channels * esize % 16 == 0 && wide_rows(x, x_ld) && wide_rows(gates, gates_ld) && wide_rows(out, channels) && reinterpret_cast<uintptr_t>(state) % 32 == 0 &&
                    reinterpret_cast<uintptr_t>(state_out) % 32 == 0;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    constexpr int V = 16 / (int)sizeof(T);
    const int per = wide ? V : 1;
    auto kernel = wide ? step_kernel<T, V> : step_kernel<T, 1>;
    D3D_LAUNCH(true, kernel, (unsigned)stream_grid(rows * (channels / per), 256), 256, 0, st, (const T*)x, x_ld, (const T*)gates, gates_ld,
               state, state_out, (T*)out, rows, channels);
    return D3D_OK;
  });
}
