// Layer norm over the channels of voxel rows, its backward pass, and rows in 8-bit integers.
//   t = x + r,  y = (t - mean) rstd w + b,  rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - <g> - xhat <g xhat>),  g = dy w,  xhat = (t - mean) rstd,  dw = sum dy xhat,  db = sum dy
//   s = max |y| / 127,  q = rint(y / s)
// All of them move bytes: every tensor is read and written once, in 16-byte pieces, a row stays in the registers of
// the threads that share it, and mean, variance and the two means of the backward pass are sums in 32 bits over those
// registers (the variance of differences to the mean, not a difference of two large sums).
// Measured, of the 6.55 TB/s that a copy gets: a norm with a residual of 120 k x 128 bf16 20.9 us, 5.9 TB/s; norm and backward pass
// of 238 k x 64 bf16 13.4 + 27.5 + 5.5 us (five passes over the rows, some of them from L2), of 4099 x 4096 in 32 bits 22 + 36 +
// 7 us; a norm of 66 k x 256 bf16 with a residual in 8 bits 28 us, 4.2 TB/s of 118 MB: neither the bytes nor the instructions (2.0 a
// cycle of 4) are all there can be; a row is a chain of three sums and the rounding, with 24 warps an SM to hide it.
// Not all fits the registers: spilled are 96 to 136 bytes a thread backward for 16-bit rows of 8 to 1024 channels (80 registers, for
// three CTAs an SM), 200 to 570 for the longest rows, 50 to 70 forward for up to 512 channels in 32 bits, 16 in 8 bits.
#include <type_traits>

#include "common.cuh"
#include "packed.cuh"

namespace d3d {
namespace {

struct NormArgs {
  const void *x, *residual;
  int64_t x_ld, residual_ld;
  const float *weight, *bias;
  float eps;
  int64_t rows;
  int channels;
  const int32_t* num_rows;  // live rows on the device, or null
  void *total, *out;        // [rows][channels]
  float *mean, *rstd;
  int8_t* q;
  int64_t q_ld;
  float* scales;
};

struct Add {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
// The larger one, NaN where either is NaN.
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
  }
};

// Threads of a CTA: several rows side by side where a row has fewer.
template <int kLanes> __host__ __device__ constexpr int threads_for() { return kLanes <= 256 ? 256 : kLanes; }

// Combines N values over the kLanes threads that share a row; every thread gets the results.  Within a warp by shuffles, beyond
// it through `scratch` (two buffers of N words a warp, used in turn: one barrier per call).
template <int kLanes, int N, class T, class Op>
__device__ __forceinline__ void row_reduce(T (&v)[N], Op op, uint32_t* scratch, int& turn) {
#pragma unroll
  for (int d = (kLanes < 32 ? kLanes : 32) / 2; d >= 1; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], d));
  if (kLanes > 32) {
    constexpr int kWarps = threads_for<kLanes>() / 32, kOfRow = kLanes > 32 ? kLanes / 32 : 1;
    T* s = reinterpret_cast<T*>(scratch) + turn * (kWarps * N);
    turn ^= 1;
    if (lane_id() == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[(threadIdx.x >> 5) * N + i] = v[i];
    __syncthreads();
    s += threadIdx.x / kLanes * kOfRow * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = s[i];
#pragma unroll
      for (int w = 1; w < kOfRow; ++w) v[i] = op(v[i], s[w * N + i]);
    }
  }
}
template <int kLanes, class T, class Op> __device__ __forceinline__ T row_reduce(T v, Op op, uint32_t* scratch, int& turn) {
  T one[1] = {v};
  row_reduce<kLanes>(one, op, scratch, turn);
  return one[0];
}

// The integer nearest to v / s, ties to even, as if the quotient were exact: the product with 1 / s is at most one step
// off, and what is left over, v - r s, has no rounding error near the border (s / 2) that decides.
__device__ __forceinline__ int nearest_step(float v, float s, float inv) {
  float r = rintf(v * inv);
  const float left = fmaf(-r, s, v), half = 0.5f * s;
  const bool odd = ((int)r & 1) != 0;
  if (left > half || (odd && left == half)) r += 1.f;
  else if (left < -half || (odd && left == -half)) r -= 1.f;
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}
// V of them.  1.5 2^23 added leaves the nearest integer in the low bits of the sum.  Where what is left over of every value is
// less than half a step, that is all; values on a border or next to it are looked at one by one.
template <int V> __device__ __forceinline__ Pack<int8_t, V> steps_of(const Vec<V>& v, float s, float inv) {
  const Vec<V> magic = all<V>(12582912.f);
  const Vec<V> sum = fma(v, all<V>(inv), magic), r = add(sum, all<V>(-12582912.f)), left = fma(r, all<V>(-s), v);
  float most = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) most = fmaxf(most, fabsf(left.v[e]));
  Pack<int8_t, V> q;
  if (most < 0.5f * s) {
#pragma unroll
    for (int e = 0; e < V; ++e) q.v[e] = (int8_t)__float_as_int(sum.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) q.v[e] = inv == 0.f ? (int8_t)0 : (int8_t)nearest_step(v.v[e], s, inv);
  }
  return q;
}
// Scale of a row with this largest magnitude.  A row that is not finite has no scale (NaN, which every product with it
// becomes), one below 127 times the smallest normal number counts as zeros; `inv` is 0 for both.
__device__ __forceinline__ float step_of(float amax, float* inv) {
  *inv = 0.f;
  if (!(amax < __uint_as_float(0x7f800000u))) return __uint_as_float(0x7fc00000u);
  const float s = __fdiv_rn(amax, 127.f);
  if (s < 1.17549435e-38f) return 0.f;
  *inv = __frcp_rn(s);
  return s;
}

// CTAs to an SM.  What counts is how much is on its way, so three, and fewer where the registers would not do: forward where the
// parameters are in them, backward for 32-bit rows (238 k x 64 bf16, backward alone, with two CTAs / three: 30.1 / 27.5 us).  Of the
// longest rows one, but forward two where they are read an element at a time (3574 x 2377 in 32 bits, one / two: 62 / 41 us).
template <int V, int kLanes> constexpr int ctas_for(bool backward) { return kLanes > 256 ? (backward || V > 1 ? 1 : 2) : (backward ? V == 4 : kLanes > 32) ? 2 : 3; }
constexpr int kMostBackwardCtas = 3 * kNumSMs;

// A thread's pieces of the rows of a tensor that it has part in, the next ones on their way while one is summed up.  The backward
// pass has two of them in turn, each for every other row.
template <class T, int V, int kVecs, int kLanes> struct Stream {
  const T* at;
  int64_t step;
  Pack<T, V> next[kVecs];
  // first: the first row of these, `stride` rows in front of the next one
  __device__ __forceinline__ Stream(const void* p, int64_t ld, int64_t first, int64_t stride, int lane)
      : at((const T*)p + first * ld + lane * V), step(stride * ld) {}
  __device__ __forceinline__ void load(bool has, int lane, int channels) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      if (has && (k * kLanes + lane) * V < channels) {
        next[k] = *reinterpret_cast<const Pack<T, V>*>(at + k * kLanes * V);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) next[k].v[e] = from_f32<T>(0.f);
      }
    }
    at += step;
  }
};
template <int V> __device__ __forceinline__ float across(const Vec<V>& x) {
  float s = x.v[0];
#pragma unroll
  for (int e = 1; e < V; ++e) s += x.v[e];
  return s;
}
// A parameter of a thread's columns, zeros behind the last one.  Where rows are long the thread has them in registers, where
// several rows share a warp they are in shared memory: the registers are better spent on rows that are on their way.
template <int V, int kVecs, int kLanes> struct Columns {
  static constexpr bool kShared = kLanes <= 32;
  static constexpr int kWidth = kShared ? V * kVecs * kLanes : 1;
  using Store = float[kWidth];
  Vec<V> held[kShared ? 1 : kVecs];
  const float* store;
  // The caller's barrier before the first use.
  __device__ __forceinline__ Columns(Store& shared, const float* p, float without, int lane, int channels) : store(shared) {
    if constexpr (kShared) {
      for (int c = threadIdx.x; c < kWidth; c += threads_for<kLanes>()) shared[c] = c >= channels ? 0.f : p ? load_fresh(p + c) : without;
    } else {
#pragma unroll
      for (int k = 0; k < kVecs; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = (k * kLanes + lane) * V + e;
          held[k].v[e] = c >= channels ? 0.f : p ? load_fresh(p + c) : without;
        }
    }
  }
  __device__ __forceinline__ Vec<V> at(int k, int lane) const {
    if constexpr (kShared) {
      Vec<V> r;
      constexpr int kStep = V < 4 ? 1 : 4;
#pragma unroll
      for (int e = 0; e < V; e += kStep) {
        const float* p = store + (k * kLanes + lane) * V + e;
        if constexpr (kStep == 4) {
          const float4 t = *reinterpret_cast<const float4*>(p);
          r.v[e] = t.x, r.v[e + 1] = t.y, r.v[e + 2] = t.z, r.v[e + 3] = t.w;
        } else {
          r.v[e] = *p;
        }
      }
      return r;
    } else {
      return held[k];
    }
  }
};

// kLanes threads share a row, kVecs pieces of V elements each.  CTAs walk over the rows, so that weight and bias are fetched once
// per CTA.
template <class T, int V, int kVecs, int kLanes, bool kNorm, bool kQuant>
__global__ void __launch_bounds__(threads_for<kLanes>(), ctas_for<V, kLanes>(false))
norm_kernel(const NormArgs a) {
  constexpr int kGroups = threads_for<kLanes>() / kLanes;
  using P = Pack<T, V>;
  __shared__ uint32_t scratch[kLanes > 32 ? 2 * (threads_for<kLanes>() / 32) : 1];
  int turn = 0;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int channels = a.channels;
  pdl_wait();  // and no early release: the next kernel's CTAs would come in between these (238 k x 64, both ways: 41 / 48 us)
  const int64_t rows = live_rows(a.rows, a.num_rows);
  const float inv_n = 1.f / (float)channels;
  const bool sum = kNorm && a.residual != nullptr;
  const int64_t stride = (int64_t)gridDim.x * kGroups;
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  const int64_t over = rows + group;  // row < over: one of the CTA's rows is there
  Stream<T, V, kVecs, kLanes> in(a.x, a.x_ld, row, stride, lane), more(a.residual, a.residual_ld, row, stride, lane);
  auto load = [&](int64_t at) {
    in.load(at < rows, lane, channels);
    if (sum) more.load(at < rows, lane, channels);
  };
  load(row);
  using Col = Columns<V, kVecs, kLanes>;
  __shared__ __align__(16) typename Col::Store w_store, b_store;
  const Col w(w_store, a.weight, 1.f, lane, kNorm ? channels : 0), b(b_store, a.bias, 0.f, lane, kNorm ? channels : 0);
  if (Col::kShared) __syncthreads();
  for (; row < over; row += stride) {
    const bool has = row < rows;
    Vec<V> y[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * kLanes + lane) * V;
      if (sum) {
        const P t = narrow<T, V>(add(widen<T, V>(in.next[k]), widen<T, V>(more.next[k])));
        if (has && c < channels) *reinterpret_cast<P*>((T*)a.total + row * channels + c) = t;
        y[k] = widen<T, V>(t);  // the norm is that of the rounded sum, which is what the backward pass will see
      } else {
        y[k] = widen<T, V>(in.next[k]);
      }
    }
    load(row + stride);
    if (kNorm) {
      Vec<V> s = y[0];
#pragma unroll
      for (int k = 1; k < kVecs; ++k) s = add(s, y[k]);
      const float mean = row_reduce<kLanes>(across(s), Add(), scratch, turn) * inv_n;
      s = all<V>(0.f);
#pragma unroll
      for (int k = 0; k < kVecs; ++k)
        if ((k * kLanes + lane) * V < channels) {
          y[k] = add(y[k], all<V>(-mean));
          s = fma(y[k], y[k], s);
        }
      const float rstd = rsqrtf(row_reduce<kLanes>(across(s), Add(), scratch, turn) * inv_n + a.eps);
      if (lane == 0 && has && a.mean) a.mean[row] = mean, a.rstd[row] = rstd;
#pragma unroll
      for (int k = 0; k < kVecs; ++k) y[k] = fma(mul(y[k], all<V>(rstd)), w.at(k, lane), b.at(k, lane));
    }
    float inv = 0.f, scale = 0.f;
    if (kQuant) {
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < kVecs; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) amax = Max()(amax, fabsf(y[k].v[e]));
      scale = step_of(row_reduce<kLanes>(amax, Max(), scratch, turn), &inv);
      if (lane == 0 && has) a.scales[row] = scale;
    }
    if (!has) continue;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * kLanes + lane) * V;
      if (c >= channels) continue;
      if (kQuant) *reinterpret_cast<Pack<int8_t, V>*>(a.q + row * a.q_ld + c) = steps_of<V>(y[k], scale, inv);
      else *reinterpret_cast<P*>((T*)a.out + row * channels + c) = narrow<T, V>(y[k]);
    }
  }
}

// Sums of the columns that a CTA of the backward pass adds up in shared memory: of its warps, or of its rows where those are longer.
template <int kLanes> __host__ __device__ constexpr int parts_for() { return threads_for<kLanes>() / (kLanes < 32 ? 32 : kLanes); }

struct NormBackwardArgs {
  const void *grad, *x, *grad_total;
  int64_t grad_ld, x_ld, grad_total_ld;
  const float *weight, *mean, *rstd;
  int64_t rows;
  int channels;
  const int32_t* num_rows;
  void* grad_x;
  float* partial;  // [CTAs][2][channels]
  float *grad_weight, *grad_bias;
};

// As above; a thread adds up the weight's and the bias's gradient of its columns over all its rows, the CTA adds its
// threads' sums in a fixed order.
template <class T, int V, int kVecs, int kLanes>
__global__ void __launch_bounds__(threads_for<kLanes>(), ctas_for<V, kLanes>(true))
norm_backward_kernel(const NormBackwardArgs a) {
  constexpr int kThreads = threads_for<kLanes>(), kGroups = kThreads / kLanes;
  using P = Pack<T, V>;
  __shared__ uint32_t scratch[kLanes > 32 ? 4 * (threads_for<kLanes>() / 32) : 1];
  extern __shared__ float sums[];  // [kParts][2][channels] where several rows share the CTA
  int turn = 0;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int channels = a.channels;
  pdl_wait();
  const int64_t rows = live_rows(a.rows, a.num_rows);
  const float inv_n = 1.f / (float)channels;
  const int64_t stride = (int64_t)gridDim.x * kGroups;
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  const int64_t over = rows + group;
  using S = Stream<T, V, kVecs, kLanes>;
  S in[2] = {S(a.x, a.x_ld, row, 2 * stride, lane), S(a.x, a.x_ld, row + stride, 2 * stride, lane)};
  S grad[2] = {S(a.grad, a.grad_ld, row, 2 * stride, lane), S(a.grad, a.grad_ld, row + stride, 2 * stride, lane)};
  float next_mean[2], next_rstd[2];
  auto load = [&](auto which, int64_t at) {
    constexpr int I = decltype(which)::value;
    const bool has = at < rows;
    in[I].load(has, lane, channels);
    grad[I].load(has, lane, channels);
    next_mean[I] = has ? load_fresh(a.mean + at) : 0.f, next_rstd[I] = has ? load_fresh(a.rstd + at) : 0.f;
  };
  load(std::integral_constant<int, 0>(), row);
  load(std::integral_constant<int, 1>(), row + stride);
  using Col = Columns<V, kVecs, kLanes>;
  __shared__ __align__(16) typename Col::Store w_store;
  const Col w(w_store, a.weight, 1.f, lane, channels);
  if (Col::kShared) __syncthreads();
  Vec<V> dw[kVecs], db[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) dw[k] = db[k] = all<V>(0.f);
  auto one = [&](auto which) {
    constexpr int I = decltype(which)::value;
    const float rstd = next_rstd[I], shift = -next_mean[I] * rstd;
    P x[kVecs], g[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) x[k] = in[I].next[k], g[k] = grad[I].next[k];
    load(which, row + 2 * stride);
    Vec<V> s1 = all<V>(0.f), s2 = all<V>(0.f);
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      // beyond the last channel gradient and weight are zeros, so xhat may be anything finite there
      const Vec<V> hat = fma(widen<T, V>(x[k]), all<V>(rstd), all<V>(shift)), dy = widen<T, V>(g[k]), gw = mul(dy, w.at(k, lane));
      s1 = add(s1, gw), s2 = fma(gw, hat, s2);
      dw[k] = fma(dy, hat, dw[k]), db[k] = add(db[k], dy);
    }
    float dot[2] = {across(s1), across(s2)};
    row_reduce<kLanes>(dot, Add(), scratch, turn);
    if (row >= rows) return;
    // rstd (g - m1 - hat m2) with hat = x rstd + shift
    const float m1 = dot[0] * inv_n, m2 = dot[1] * inv_n;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int c = (k * kLanes + lane) * V;
      if (c >= channels) continue;
      const Vec<V> hat = fma(widen<T, V>(x[k]), all<V>(rstd), all<V>(shift));
      Vec<V> d = fma(widen<T, V>(g[k]), w.at(k, lane), fma(hat, all<V>(-m2), all<V>(-m1)));
      d = mul(d, all<V>(rstd));
      if (a.grad_total) d = add(d, widen<T, V>(*reinterpret_cast<const P*>((const T*)a.grad_total + row * a.grad_total_ld + c)));
      *reinterpret_cast<P*>((T*)a.grad_x + row * channels + c) = narrow<T, V>(d);
    }
  };
  while (row < over) {
    one(std::integral_constant<int, 0>());
    row += stride;
    if (row >= over) break;
    one(std::integral_constant<int, 1>());
    row += stride;
  }
  float* mine = a.partial + (int64_t)blockIdx.x * 2 * channels;
  float* mine_b = mine + channels;
  if (gridDim.x == 1) mine = a.grad_weight, mine_b = a.grad_bias;  // the only CTA's sums are the result
  if (kGroups > 1) {  // the groups of a warp by shuffles, the others through shared memory
    constexpr int kParts = parts_for<kLanes>();
    float* part = sums + (kLanes < 32 ? threadIdx.x >> 5 : group) * 2 * channels;
#pragma unroll
    for (int d = 16; d >= kLanes; d >>= 1)
#pragma unroll
      for (int k = 0; k < kVecs; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          dw[k].v[e] += __shfl_xor_sync(0xffffffffu, dw[k].v[e], d);
          db[k].v[e] += __shfl_xor_sync(0xffffffffu, db[k].v[e], d);
        }
    if (kLanes >= 32 || lane_id() < kLanes)
#pragma unroll
      for (int k = 0; k < kVecs; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = (k * kLanes + lane) * V + e;
          if (c < channels) part[c] = dw[k].v[e], part[channels + c] = db[k].v[e];
        }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * channels; c += kThreads) {
      float t = sums[c];
#pragma unroll
      for (int i = 1; i < kParts; ++i) t += sums[i * 2 * channels + c];
      float* to = c < channels ? mine : mine_b;
      if (to) to[c < channels ? c : c - channels] = t;
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = (k * kLanes + lane) * V + e;
        if (c < channels && mine) mine[c] = dw[k].v[e];
        if (c < channels && mine_b) mine_b[c] = db[k].v[e];
      }
  }
}

// Sums the CTAs' partial gradients in a fixed order: eight columns to a CTA, 64 threads of each take the partials in turn.
__global__ void __launch_bounds__(512)
norm_columns_kernel(const float* partial, int parts, int channels, float* __restrict__ grad_weight,
                    float* __restrict__ grad_bias) {
  __shared__ float s[16][8];
  pdl_release();
  pdl_wait();
  const int lane = lane_id(), warp = threadIdx.x >> 5, c = blockIdx.x * 8 + lane % 8;
  float sum = 0.f;
  if (c < 2 * channels)
#pragma unroll 8
    for (int p = threadIdx.x / 8; p < parts; p += 64) sum += __ldcg(partial + (int64_t)p * 2 * channels + c);
  sum += __shfl_xor_sync(0xffffffffu, sum, 8);
  sum += __shfl_xor_sync(0xffffffffu, sum, 16);
  if (lane < 8) s[warp][lane] = sum;
  __syncthreads();
  if (threadIdx.x < 8 && c < 2 * channels) {
    float t = s[0][lane];
#pragma unroll
    for (int w = 1; w < 16; ++w) t += s[w][lane];
    if (c < channels) {
      if (grad_weight) grad_weight[c] = t;
    } else if (grad_bias) grad_bias[c - channels] = t;
  }
}

constexpr int kMaxChannels = 8192;

// f(elements of a piece, pieces, threads of a row) for the shape that covers the channels: K pieces a thread up to 512 threads.
template <int V, int K, class F> int by_shape(int channels, F f) {
#define D3D_NORM_SHAPE(K, L) return f(std::integral_constant<int, V>(), std::integral_constant<int, K>(), std::integral_constant<int, L>())
  const int n = (channels + V * K - 1) / (V * K);
  if constexpr (V > 1) {
    if (n <= 1) D3D_NORM_SHAPE(K, 1);
  }
  if (n <= 2) D3D_NORM_SHAPE(K, 2);
  if (n <= 4) D3D_NORM_SHAPE(K, 4);
  if (n <= 8) D3D_NORM_SHAPE(K, 8);
  if (n <= 16) D3D_NORM_SHAPE(K, 16);
  if (n <= 32) D3D_NORM_SHAPE(K, 32);
  if (n <= 64) D3D_NORM_SHAPE(K, 64);
  if (n <= 128) D3D_NORM_SHAPE(K, 128);
  if (n <= 256) D3D_NORM_SHAPE(K, 256);
  if (n <= 512 || V * K >= 16) D3D_NORM_SHAPE(K, 512);
  if constexpr (V * K < 16) D3D_NORM_SHAPE(16 / V, 512);
  return D3D_ERR_TOO_LARGE;
#undef D3D_NORM_SHAPE
}

// Sixteen elements a thread, which keeps what the sums cost small; eight in the backward pass, where a thread has the columns' sums
// beside them.  Rows that cannot be read in pieces: one element at a time,
// four or eight of a thread (18.5 k rows of 131 in 8 bits, four / eight: 10.0 / 8.3 us).
template <class T, bool kBackward, class F> int by_alignment(bool wide, int channels, F f) {
  constexpr int V = 16 / (int)sizeof(T), K = (kBackward ? 8 : 16) / V;
  return wide ? by_shape<V, K>(channels, f) : by_shape<1, kBackward ? 4 : 8>(channels, f);
}
template <class F> int by_type(int dtype, F f) {
  switch (dtype) {
    case D3D_FLOAT: return f(float());
    case D3D_HALF: return f(__half());
    case D3D_BF16: return f(__nv_bfloat16());
    default: return D3D_ERR_UNSUPPORTED_DTYPE;
  }
}

// Whether rows of `ld` elements from `p` on can be read in 16-byte pieces.
bool rows_wide(const void* p, int64_t ld, int esize) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * esize % 16 == 0;
}

// CTAs of `kernel` that fill the GPU once.
template <class K> int resident(K kernel, int threads, size_t smem) {
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) n = 1;
  return n * kNumSMs;
}

template <bool kNorm, bool kQuant> int launch_norm(int dtype, bool wide, const NormArgs& a, cudaStream_t st) {
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return by_alignment<T, false>(wide, a.channels, [&](auto v, auto k, auto l) -> int {
      constexpr int V = decltype(v)::value, K = decltype(k)::value, L = decltype(l)::value;
      constexpr int per_cta = threads_for<L>() / L;
      auto kernel = norm_kernel<T, V, K, L, kNorm, kQuant>;
      static const int most = resident(kernel, threads_for<L>(), 0);
      const int64_t need = ceil_div(a.rows, per_cta);
      D3D_LAUNCH(true, kernel, (unsigned)(need < most ? need : most), threads_for<L>(), 0, st, a);
      return D3D_OK;
    });
  });
}

// The backward pass keeps its sums per CTA, so that their number decides how large the workspace is: one wave of them.
int backward_ctas(int64_t rows, int per_cta, int64_t most) {
  const int64_t need = ceil_div(rows > 0 ? rows : 1, per_cta);
  return (int)(need < most ? need : most);
}

}  // namespace
}  // namespace d3d

using namespace d3d;

extern "C" int d3d_layer_norm(int dtype, const void* x, int64_t x_ld, const void* residual, int64_t residual_ld,
                              const float* weight, const float* bias, float eps, int64_t rows, int channels,
                              const int32_t* num_rows, void* total, void* out, float* mean, float* rstd, void* stream) {
  D3D_NVTX_RANGE("d3d_layer_norm");
  const int esize = (int)dtype_size(dtype);
  D3D_REQUIRE(dtype == D3D_FLOAT || dtype == D3D_HALF || dtype == D3D_BF16, D3D_ERR_UNSUPPORTED_DTYPE);
  D3D_REQUIRE(rows >= 0 && channels >= 1 && eps >= 0.f && x_ld >= channels && (!residual || residual_ld >= channels) &&
                  !residual == !total && !mean == !rstd,
              D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(channels <= kMaxChannels, D3D_ERR_TOO_LARGE);
  if (rows == 0) return D3D_OK;
  D3D_REQUIRE(x && out && on_multiples(esize, x, residual, out, total) && on_multiples(4, weight, bias, num_rows, mean, rstd),
              D3D_ERR_INVALID_ARGUMENT);
  NormArgs a = {};
  a.x = x, a.x_ld = x_ld, a.residual = residual, a.residual_ld = residual_ld, a.weight = weight, a.bias = bias, a.eps = eps;
  a.rows = rows, a.channels = channels, a.num_rows = num_rows, a.total = total, a.out = out, a.mean = mean, a.rstd = rstd;
  const bool wide = channels * esize % 16 == 0 && rows_wide(x, x_ld, esize) && (!residual || rows_wide(residual, residual_ld, esize)) &&
                    rows_wide(out, channels, esize) && rows_wide(total, channels, esize);
  return launch_norm<true, false>(dtype, wide, a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int d3d_layer_norm_int8(int dtype, const void* x, int64_t x_ld, const void* residual, int64_t residual_ld,
                                   const float* weight, const float* bias, float eps, int64_t rows, int channels,
                                   const int32_t* num_rows, void* total, int8_t* q, int64_t q_ld, float* scales,
                                   void* stream) {
  D3D_NVTX_RANGE("d3d_layer_norm_int8");
  const int esize = (int)dtype_size(dtype);
  D3D_REQUIRE(dtype == D3D_FLOAT || dtype == D3D_HALF || dtype == D3D_BF16, D3D_ERR_UNSUPPORTED_DTYPE);
  D3D_REQUIRE(rows >= 0 && channels >= 1 && eps >= 0.f && x_ld >= channels && (!residual || residual_ld >= channels) &&
                  !residual == !total && q_ld >= channels,
              D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(channels <= kMaxChannels, D3D_ERR_TOO_LARGE);
  if (rows == 0) return D3D_OK;
  D3D_REQUIRE(x && q && scales && on_multiples(esize, x, residual, total) && on_multiples(4, weight, bias, num_rows, scales),
              D3D_ERR_INVALID_ARGUMENT);
  NormArgs a = {};
  a.x = x, a.x_ld = x_ld, a.residual = residual, a.residual_ld = residual_ld, a.weight = weight, a.bias = bias, a.eps = eps;
  a.rows = rows, a.channels = channels, a.num_rows = num_rows, a.total = total, a.q = q, a.q_ld = q_ld, a.scales = scales;
  const bool wide = channels * esize % 16 == 0 && rows_wide(x, x_ld, esize) && (!residual || rows_wide(residual, residual_ld, esize)) &&
                    rows_wide(total, channels, esize) && reinterpret_cast<uintptr_t>(q) % 8 == 0 && q_ld % 8 == 0;
  return launch_norm<true, true>(dtype, wide, a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int d3d_quantize_rows(int dtype, const void* x, int64_t x_ld, int64_t rows, int channels, const int32_t* num_rows,
                                 int8_t* q, int64_t q_ld, float* scales, void* stream) {
  D3D_NVTX_RANGE("d3d_quantize_rows");
  const int esize = (int)dtype_size(dtype);
  D3D_REQUIRE(dtype == D3D_FLOAT || dtype == D3D_HALF || dtype == D3D_BF16, D3D_ERR_UNSUPPORTED_DTYPE);
  D3D_REQUIRE(rows >= 0 && channels >= 1 && x_ld >= channels && q_ld >= channels, D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(channels <= kMaxChannels, D3D_ERR_TOO_LARGE);
  if (rows == 0) return D3D_OK;
  D3D_REQUIRE(x && q && scales && on_multiples(esize, x) && on_multiples(4, num_rows, scales), D3D_ERR_INVALID_ARGUMENT);
  NormArgs a = {};
  a.x = x, a.x_ld = x_ld, a.rows = rows, a.channels = channels, a.num_rows = num_rows, a.q = q, a.q_ld = q_ld, a.scales = scales;
  const bool wide = channels * esize % 16 == 0 && rows_wide(x, x_ld, esize) && reinterpret_cast<uintptr_t>(q) % 8 == 0 && q_ld % 8 == 0;
  return launch_norm<false, true>(dtype, wide, a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t d3d_layer_norm_backward_workspace(int64_t rows, int channels) {
  if (rows < 0 || channels < 1) return 0;
  return (size_t)backward_ctas(rows, 1, kMostBackwardCtas) * 2 * channels * sizeof(float);
}

extern "C" int d3d_layer_norm_backward(int dtype, const void* grad, int64_t grad_ld, const void* x, int64_t x_ld,
                                       const void* grad_total, int64_t grad_total_ld, const float* weight, const float* mean,
                                       const float* rstd, int64_t rows, int channels, const int32_t* num_rows, void* grad_x,
                                       float* grad_weight, float* grad_bias, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  D3D_NVTX_RANGE("d3d_layer_norm_backward");
  const int esize = (int)dtype_size(dtype);
  D3D_REQUIRE(dtype == D3D_FLOAT || dtype == D3D_HALF || dtype == D3D_BF16, D3D_ERR_UNSUPPORTED_DTYPE);
  D3D_REQUIRE(rows >= 0 && channels >= 1 && x_ld >= channels && grad_ld >= channels && (!grad_total || grad_total_ld >= channels),
              D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(channels <= kMaxChannels, D3D_ERR_TOO_LARGE);
  D3D_REQUIRE(rows == 0 || (x && grad && mean && rstd && grad_x), D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(on_multiples(esize, x, grad, grad_total, grad_x) && on_multiples(4, weight, mean, rstd, num_rows, grad_weight, grad_bias),
              D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace && on_multiples(4, workspace), D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace_bytes >= d3d_layer_norm_backward_workspace(rows, channels), D3D_ERR_WORKSPACE_TOO_SMALL);
  NormBackwardArgs a = {};
  a.grad = grad, a.grad_ld = grad_ld, a.x = x, a.x_ld = x_ld, a.grad_total = grad_total, a.grad_total_ld = grad_total_ld;
  a.weight = weight, a.mean = mean, a.rstd = rstd, a.rows = rows, a.channels = channels, a.num_rows = num_rows, a.grad_x = grad_x;
  a.partial = reinterpret_cast<float*>(workspace), a.grad_weight = grad_weight, a.grad_bias = grad_bias;
  const bool wide = channels * esize % 16 == 0 && rows_wide(x, x_ld, esize) && rows_wide(grad, grad_ld, esize) &&
                    (!grad_total || rows_wide(grad_total, grad_total_ld, esize)) && rows_wide(grad_x, channels, esize);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return by_alignment<T, true>(wide, channels, [&](auto v, auto k, auto l) -> int {
      constexpr int V = decltype(v)::value, K = decltype(k)::value, L = decltype(l)::value;
      constexpr int per_cta = threads_for<L>() / L;
      const int ctas = backward_ctas(rows, per_cta, ctas_for<V, L>(true) * kNumSMs);
      const size_t smem = threads_for<L>() > L ? (size_t)parts_for<L>() * 2 * channels * sizeof(float) : 0;
      D3D_LAUNCH(true, (norm_backward_kernel<T, V, K, L>), (unsigned)ctas, threads_for<L>(), smem, st, a);
      if (ctas > 1)
        D3D_LAUNCH(true, norm_columns_kernel, (unsigned)ceil_div(2 * channels, 8), 512, 0, st, a.partial, ctas, channels, grad_weight,
                   grad_bias);
      return D3D_OK;
    });
  });
}
