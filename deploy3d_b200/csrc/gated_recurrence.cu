// Gated linear recurrence over sequences of voxel rows, its backward pass, and its form for one row a sequence.
//   h[t] = f[t] h[t-1] + (1 - f[t]) x[t],  f = sigmoid(gate);  h in front of a sequence is initial[s] (zeros without)
//   delta[t] = grad[t] + f[t+1] delta[t+1]  (+ grad_final[s] at the last row),  dx = delta (1 - f),
//   dgate = delta (h[t-1] - x) f (1 - f),  dinitial[s] = f delta at the first row
// A step is the map c -> a c + b.  Maps compose: (a2, b2) after (a1, b1) is (a2 a1, a2 b1 + b2), so a tile of rows is one map
// per channel, and tiles can be worked on side by side.  A row that starts a sequence is the map c -> b whatever c is, also
// where c is not finite: its a is -0, and the sign says that what came before is not looked at (products keep it, f is never
// negative).
// Everything is held in 32 bits; 1 - f is computed as sigmoid(-gate), not as a difference, and f as 1 - (1 - f) where it is
// the larger one, so that neither loses digits at long memories.
#include <type_traits>

#include "common.cuh"

namespace d3d {
namespace {

template <class T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// Rows of a tile, whatever the types: the states the forward pass leaves at their starts are those of the backward pass.
constexpr int kTile = 128;
__host__ __device__ constexpr int backward_threads(int lanes) { return lanes >= 8 ? 512 : 256; }

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

// f and 1 - f
__device__ __forceinline__ void gate_of(float g, float* f, float* add) {
  const float e = expf(-fabsf(g)), small = e * __fdividef(1.f, 1.f + e), large = 1.f - small;
  *f = fabsf(g >= 0.f ? large : small);  // NaN without a sign: the sign of a map means a reset
  *add = g >= 0.f ? small : large;
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
// The sequence row t belongs to: the last one that starts at or before it.
__device__ __forceinline__ int seq_of(const ScanArgs& a, int64_t t) {
  int lo = 0, hi = a.seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.offsets + mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// For the rows of a tile, in the order they are walked in: the sequence that starts / ends there, or -1.
template <int kThreads>
__device__ __forceinline__ void mark_ends(const ScanArgs& a, const Span& span, int tile, int* first, int* last) {
  for (int i = threadIdx.x; i < kTile; i += kThreads) {
    const int64_t p = (int64_t)tile * kTile + i;
    int f = -1, l = -1;
    if (p < span.count) {
      const int64_t t = row_at(a, span, p);
      const int s = seq_of(a, t);
      const bool at_low = t == __ldg(a.offsets + s), at_high = t + 1 == __ldg(a.offsets + s + 1);
      f = (a.reverse ? at_high : at_low) ? s : -1;
      l = (a.reverse ? at_low : at_high) ? s : -1;
    }
    first[i] = f, last[i] = l;
  }
}

// Every thread has a map per channel; afterwards it has that of all threads in front of it (kUp) or behind it.  kLanes lanes
// of a warp stand side by side along the channels.  totals: [2][kWarps][kLanes * V], left with the warps' maps.
template <int kLanes, int V, int kWarps, bool kUp>
__device__ __forceinline__ void scan_threads(float (&a)[V], float (&b)[V], float* totals) {
  const int lane = lane_id(), warp = threadIdx.x >> 5, at = lane % kLanes * V;
  constexpr int kWidth = kLanes * V;
#pragma unroll
  for (int d = kLanes; d < 32; d <<= 1)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float pa = kUp ? __shfl_up_sync(0xffffffffu, a[e], d) : __shfl_down_sync(0xffffffffu, a[e], d);
      const float pb = kUp ? __shfl_up_sync(0xffffffffu, b[e], d) : __shfl_down_sync(0xffffffffu, b[e], d);
      if ((kUp ? lane >= d : lane + d < 32) && !is_reset(a[e])) b[e] = fmaf(a[e], pb, b[e]), a[e] *= pa;
    }
  if (kUp ? lane >= 32 - kLanes : lane < kLanes)
#pragma unroll
    for (int e = 0; e < V; ++e) totals[warp * kWidth + at + e] = a[e], totals[(kWarps + warp) * kWidth + at + e] = b[e];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float pa = kUp ? __shfl_up_sync(0xffffffffu, a[e], kLanes & 31) : __shfl_down_sync(0xffffffffu, a[e], kLanes & 31);
    const float pb = kUp ? __shfl_up_sync(0xffffffffu, b[e], kLanes & 31) : __shfl_down_sync(0xffffffffu, b[e], kLanes & 31);
    const bool has = kLanes < 32 && (kUp ? lane >= kLanes : lane + kLanes < 32);
    a[e] = has ? pa : 1.f, b[e] = has ? pb : 0.f;
  }
  __syncthreads();
  float pa[V], pb[V];
#pragma unroll
  for (int e = 0; e < V; ++e) pa[e] = 1.f, pb[e] = 0.f;
  for (int i = 0; i < (kUp ? warp : kWarps - 1 - warp); ++i) {
    const int w = kUp ? i : kWarps - 1 - i;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float wa = totals[w * kWidth + at + e], wb = totals[(kWarps + w) * kWidth + at + e];
      if (is_reset(wa)) pa[e] = wa, pb[e] = wb;
      else pb[e] = fmaf(wa, pb[e], wb), pa[e] *= wa;
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (!is_reset(a[e])) b[e] = fmaf(a[e], pb[e], b[e]), a[e] *= pa[e];
}
// The tile's map of the channel at `c` of its slab, from the warps' maps.
template <int kWidth, int kWarps, bool kUp> __device__ __forceinline__ float2 tile_map(const float* totals, int c) {
  float a = 1.f, b = 0.f;
  for (int i = 0; i < kWarps; ++i) {
    const int w = kUp ? i : kWarps - 1 - i;
    const float wa = totals[w * kWidth + c], wb = totals[(kWarps + w) * kWidth + c];
    if (is_reset(wa)) a = wa, b = wb;
    else b = fmaf(wa, b, wb), a *= wa;
  }
  return make_float2(a, b);
}

// A tile is kTile rows by kLanes * V channels; a thread has kRows rows of V channels in its registers.
// kMaps: the first pass, which leaves the tile's map.
template <class T, int V, int kLanes, bool kMaps>
__global__ void __launch_bounds__(256)
scan_kernel(const ScanArgs a) {
  constexpr int kThreads = 256, kRows = kTile * kLanes / kThreads, kWidth = kLanes * V, kWarps = kThreads / 32;
  using P = Pack<T, V>;
  __shared__ int first[kTile], last[kTile];
  __shared__ float totals[2 * kWarps * kWidth];
  const int slabs = (a.channels + kWidth - 1) / kWidth, slab = blockIdx.x % slabs, tile = blockIdx.x / slabs;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, c = slab * kWidth + lane * V;
  const bool live = c < a.channels;
  const Span span = span_of(a);
  P x[kRows], g[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t p = (int64_t)tile * kTile + group * kRows + r, t = row_at(a, span, p);
    if (live && p < span.count) {
      x[r] = *reinterpret_cast<const P*>((const T*)a.x + t * a.x_ld + c);
      g[r] = *reinterpret_cast<const P*>((const T*)a.gates + t * a.gates_ld + c);
    }
  }
  mark_ends<kThreads>(a, span, tile, first, last);
  __syncthreads();
  float f[kRows][V], u[kRows][V], ma[V], mb[V];
#pragma unroll
  for (int e = 0; e < V; ++e) ma[e] = 1.f, mb[e] = 0.f;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const bool in = live && (int64_t)tile * kTile + group * kRows + r < span.count;
    const int s = first[group * kRows + r];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float add;
      f[r][e] = 1.f, u[r][e] = 0.f;
      if (in) {
        gate_of(to_f32(g[r].v[e]), &f[r][e], &add);
        u[r][e] = add * to_f32(x[r].v[e]);
        if (s >= 0) {
          if (a.initial) u[r][e] = fmaf(f[r][e], __ldg(a.initial + (int64_t)s * a.channels + c + e), u[r][e]);
          f[r][e] = reset_mark();
        }
      }
      if (is_reset(f[r][e])) ma[e] = f[r][e], mb[e] = u[r][e];
      else mb[e] = fmaf(f[r][e], mb[e], u[r][e]), ma[e] *= f[r][e];
    }
  }
  scan_threads<kLanes, V, kWarps, true>(ma, mb, totals);
  if constexpr (kMaps) {
    if ((int)threadIdx.x < kWidth && slab * kWidth + (int)threadIdx.x < a.channels)
      a.maps[(int64_t)tile * a.channels + slab * kWidth + threadIdx.x] = tile_map<kWidth, kWarps, true>(totals, threadIdx.x);
    return;
  }
  float h[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float before = live && a.states ? __ldg(a.states + (int64_t)tile * a.channels + c + e) : 0.f;
    h[e] = is_reset(ma[e]) ? mb[e] : fmaf(ma[e], before, mb[e]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t p = (int64_t)tile * kTile + group * kRows + r, t = row_at(a, span, p);
    if (!live || p >= span.count) continue;
    const int s = last[group * kRows + r];
    P o;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      h[e] = is_reset(f[r][e]) ? u[r][e] : fmaf(f[r][e], h[e], u[r][e]);
      o.v[e] = from_f32<T>(h[e]);
      if (s >= 0 && a.final_state) a.final_state[(int64_t)s * a.channels + c + e] = h[e];
    }
    *reinterpret_cast<P*>((T*)a.out + t * a.channels + c) = o;
  }
}

// The tiles' maps one after the other, a thread per channel: what comes into each tile.
__global__ void __launch_bounds__(128) carry_kernel(const float2* maps, float* into, int tiles, int channels, int backward) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= channels) return;
  float h = 0.f;
  for (int i = 0; i < tiles; ++i) {
    const int64_t at = (int64_t)(backward ? tiles - 1 - i : i) * channels + c;
    into[at] = h;
    const float2 m = __ldg(maps + at);
    h = is_reset(m.x) ? m.y : fmaf(m.x, h, m.y);
  }
}

// Sequences without rows end as they start.
__global__ void __launch_bounds__(256) empty_kernel(const ScanArgs a, const float* from, float* to) {
  const int64_t n = (int64_t)a.seqs * a.channels, nth = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += nth) {
    const int64_t s = i / a.channels;
    if (__ldg(a.offsets + s + 1) <= __ldg(a.offsets + s)) to[i] = from ? __ldg(from + i) : 0.f;
  }
}

// Backward: the rows of a tile forward once more from the state in front of it, which gives h[t-1], and the gradients from its
// end.  The map of a row is c -> f (grad + c): c comes in from the row behind and goes out to the row in front.
template <class T, int V, int kLanes, bool kMaps>
__global__ void __launch_bounds__(backward_threads(kLanes))
scan_backward_kernel(const ScanArgs a) {
  constexpr int kThreads = backward_threads(kLanes), kRows = kTile * kLanes / kThreads, kWidth = kLanes * V, kWarps = kThreads / 32;
  using P = Pack<T, V>;
  __shared__ int first[kTile], last[kTile];
  __shared__ float totals[2 * kWarps * kWidth];
  const int slabs = (a.channels + kWidth - 1) / kWidth, slab = blockIdx.x % slabs, tile = blockIdx.x / slabs;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, c = slab * kWidth + lane * V;
  const bool live = c < a.channels;
  const Span span = span_of(a);
  P x[kRows], g[kRows], d[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t p = (int64_t)tile * kTile + group * kRows + r, t = row_at(a, span, p);
    if (live && p < span.count) {
      if (!kMaps) x[r] = *reinterpret_cast<const P*>((const T*)a.x + t * a.x_ld + c);
      g[r] = *reinterpret_cast<const P*>((const T*)a.gates + t * a.gates_ld + c);
      d[r] = *reinterpret_cast<const P*>((const T*)a.grad + t * a.grad_ld + c);
    }
  }
  mark_ends<kThreads>(a, span, tile, first, last);
  __syncthreads();
  float f[kRows][V], add[kRows][V], ma[V], mb[V];
  bool in[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    in[r] = live && (int64_t)tile * kTile + group * kRows + r < span.count;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      f[r][e] = 1.f, add[r][e] = 0.f;
      if (in[r]) gate_of(to_f32(g[r].v[e]), &f[r][e], &add[r][e]);
    }
  }
  float before[kRows][V];  // h[t-1]
  if (!kMaps) {
#pragma unroll
    for (int e = 0; e < V; ++e) ma[e] = 1.f, mb[e] = 0.f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (!in[r]) continue;
      const int s = first[group * kRows + r];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float u = add[r][e] * to_f32(x[r].v[e]);
        if (s >= 0) {
          const float h0 = a.initial ? __ldg(a.initial + (int64_t)s * a.channels + c + e) : 0.f;
          ma[e] = reset_mark(), mb[e] = fmaf(f[r][e], h0, u);
        } else {
          mb[e] = fmaf(f[r][e], mb[e], u), ma[e] *= f[r][e];
        }
      }
    }
    scan_threads<kLanes, V, kWarps, true>(ma, mb, totals);
    __syncthreads();
    float h[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float h0 = live ? __ldg(a.states + (int64_t)tile * a.channels + c + e) : 0.f;
      h[e] = is_reset(ma[e]) ? mb[e] : fmaf(ma[e], h0, mb[e]);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (!in[r]) continue;
      const int s = first[group * kRows + r];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (s >= 0) h[e] = a.initial ? __ldg(a.initial + (int64_t)s * a.channels + c + e) : 0.f;
        before[r][e] = h[e];
        h[e] = fmaf(f[r][e], h[e], add[r][e] * to_f32(x[r].v[e]));
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) ma[e] = 1.f, mb[e] = 0.f;
#pragma unroll
  for (int r = kRows - 1; r >= 0; --r) {
    if (!in[r]) continue;
    const int s = last[group * kRows + r];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float dy = to_f32(d[r].v[e]);
      if (s >= 0) {
        const float dl = a.grad_final ? __ldg(a.grad_final + (int64_t)s * a.channels + c + e) : 0.f;
        ma[e] = reset_mark(), mb[e] = f[r][e] * (dy + dl);
      } else {
        mb[e] = f[r][e] * (dy + mb[e]), ma[e] *= f[r][e];
      }
    }
  }
  scan_threads<kLanes, V, kWarps, false>(ma, mb, totals);
  if (kMaps) {
    if ((int)threadIdx.x < kWidth && slab * kWidth + (int)threadIdx.x < a.channels)
      a.maps[(int64_t)tile * a.channels + slab * kWidth + threadIdx.x] = tile_map<kWidth, kWarps, false>(totals, threadIdx.x);
    return;
  }
  float q[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float behind = live ? __ldg(a.carry + (int64_t)tile * a.channels + c + e) : 0.f;
    q[e] = is_reset(ma[e]) ? mb[e] : fmaf(ma[e], behind, mb[e]);
  }
#pragma unroll
  for (int r = kRows - 1; r >= 0; --r) {
    if (!in[r]) continue;
    const int64_t t = row_at(a, span, (int64_t)tile * kTile + group * kRows + r);
    const int s = last[group * kRows + r], s0 = first[group * kRows + r];
    P dx, dg;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (s >= 0) q[e] = a.grad_final ? __ldg(a.grad_final + (int64_t)s * a.channels + c + e) : 0.f;
      const float delta = to_f32(d[r].v[e]) + q[e];
      q[e] = f[r][e] * delta;
      dx.v[e] = from_f32<T>(delta * add[r][e]);
      dg.v[e] = from_f32<T>(q[e] * add[r][e] * (before[r][e] - to_f32(x[r].v[e])));
      if (s0 >= 0 && a.grad_initial) a.grad_initial[(int64_t)s0 * a.channels + c + e] = q[e];
    }
    *reinterpret_cast<P*>((T*)a.grad_x + t * a.channels + c) = dx;
    *reinterpret_cast<P*>((T*)a.grad_gates + t * a.channels + c) = dg;
  }
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
    P o;
    Pack<float, V> h;
#pragma unroll
    for (int e = 0; e < V; ++e) h.v[e] = state[at + e];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float f, add;
      gate_of(to_f32(pg.v[e]), &f, &add);
      h.v[e] = fmaf(f, h.v[e], add * to_f32(px.v[e]));
      o.v[e] = from_f32<T>(h.v[e]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) state_out[at + e] = h.v[e];
    *reinterpret_cast<P*>(out + at) = o;
  }
}

// f(V, lanes) for the tile shape of this many channels.  Rows that cannot be read in 16-byte pieces: a channel a thread.
template <class T, class F> int by_shape(bool wide, int channels, F f) {
  constexpr int V = 16 / (int)sizeof(T);
#define D3D_SCAN_SHAPE(V, L) return f(std::integral_constant<int, V>(), std::integral_constant<int, L>())
  if (!wide) D3D_SCAN_SHAPE(1, 32);
  if (channels <= 2 * V) D3D_SCAN_SHAPE(V, 2);
  if (channels <= 4 * V) D3D_SCAN_SHAPE(V, 4);
  D3D_SCAN_SHAPE(V, 8);
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

bool rows_wide(const void* p, int64_t ld, int esize) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * esize % 16 == 0; }

int fill_empty(const ScanArgs& a, const float* from, float* to, cudaStream_t st) {
  if (!to || a.seqs == 0) return D3D_OK;
  empty_kernel<<<stream_grid((int64_t)a.seqs * a.channels, 256), 256, 0, st>>>(a, from, to);
  D3D_CHECK_LAUNCH();
  return D3D_OK;
}

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
  const bool wide = channels * esize % 16 == 0 && rows_wide(x, x_ld, esize) && rows_wide(gates, gates_ld, esize) && rows_wide(out, channels, esize);
  if (seqs == 0) return D3D_OK;
  const int rc2 = fill_empty(a, initial, final_state, st);
  if (rc2 != D3D_OK || rows == 0) return rc2;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return by_shape<T>(wide, channels, [&](auto v, auto l) -> int {
      constexpr int V = decltype(v)::value, L = decltype(l)::value;
      a.tiles = (int)ceil_div(rows, kTile);
      const unsigned grid = (unsigned)(a.tiles * ceil_div(channels, L * V));
      scan_kernel<T, V, L, true><<<grid, 256, 0, st>>>(a);
      carry_kernel<<<(unsigned)ceil_div(channels, 128), 128, 0, st>>>(a.maps, a.states, a.tiles, channels, 0);
      scan_kernel<T, V, L, false><<<grid, 256, 0, st>>>(a);
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
  const bool wide = channels * esize % 16 == 0 && rows_wide(x, x_ld, esize) && rows_wide(gates, gates_ld, esize) &&
                    rows_wide(grad, grad_ld, esize) && rows_wide(grad_x, channels, esize) && rows_wide(grad_gates, channels, esize);
  if (seqs == 0) return D3D_OK;
  const int rc2 = fill_empty(a, grad_final, grad_initial, st);
  if (rc2 != D3D_OK || rows == 0) return rc2;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return by_shape<T>(wide, channels, [&](auto v, auto l) -> int {
      constexpr int V = decltype(v)::value, L = decltype(l)::value;
      a.tiles = (int)ceil_div(rows, kTile);
      const unsigned grid = (unsigned)(a.tiles * ceil_div(channels, L * V));
      scan_backward_kernel<T, V, L, true><<<grid, backward_threads(L), 0, st>>>(a);
      carry_kernel<<<(unsigned)ceil_div(channels, 128), 128, 0, st>>>(a.maps, a.carry, a.tiles, channels, 1);
      scan_backward_kernel<T, V, L, false><<<grid, backward_threads(L), 0, st>>>(a);
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
  const bool wide = channels * esize % 16 == 0 && rows_wide(x, x_ld, esize) && rows_wide(gates, gates_ld, esize) &&
                    rows_wide(out, channels, esize) && reinterpret_cast<uintptr_t>(state) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(state_out) % 16 == 0;
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
