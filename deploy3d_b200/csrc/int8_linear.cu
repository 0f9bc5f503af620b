// Product of 8-bit rows and 8-bit weights with a scale per row and per output channel:
//   out[m][n] = x_scale[m] w_scale[n] sum_k q[m][k] w[n][k] + bias[n]
// The sum is exact (32-bit integers, |sum| <= 2^14 k), the rest is three 32-bit operations and one rounding.
//
// tcgen05.mma (kind::i8, K = 32 per instruction) over tiles of 128 or, with two CTAs to a tile, 256 rows by up to 256 output
// channels: operands by TMA in 128-byte rows (128 channels of the sum a stage), several accumulators in tensor memory so that
// the epilogue of one tile runs beside the products of the next.  Up to kFewRows rows: the other way round, tiles of 128 output
// channels by all rows.  Little work is left to the integer units.
// Measured: 8192 x 4096 -> 8192 bf16 170 us, 3.2 Pop/s, the tensor cores 87 % busy (in a row of calls the power cap makes it 175 to
// 205); short sums are bound by what happens to an output piece, accumulator to registers to shared memory to memory, one after
// the other: 238 k x 64 -> 192 fp16 33 us, 3.2 TB/s, tensor cores 4 %; one row 4096 -> 4096 5.5 us, 3 TB/s of weights.
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "kernel_errors.h"
#include "packed.cuh"
#include "tc_ptx.cuh"

namespace d3d {
namespace {

__device__ int g_int8_error;  // 0 ok; otherwise the code of the first wait that gave up

struct LinearArgs {
  const int8_t *x, *w;
  int64_t x_ld, w_ld;
  const float *x_scale, *w_scale, *bias;
  void* out;
  int64_t rows;
  const int32_t* num_rows;
  int inputs, outputs;
};

// ---- little work ------------------------------------------------------------------------------------------------------
// A warp per output channel: its weights stream by once, eight pieces of a lane on their way, and are multiplied with those of kM
// rows.  kBytes: what one load takes (16 where rows start on 16 bytes, else one).
template <class T, int kM, int kBytes>
__global__ void __launch_bounds__(256)
dot_kernel(const LinearArgs a) {
  pdl_release();
  pdl_wait();
  const int64_t rows = live_rows(a.rows, a.num_rows);
  const int64_t m0 = (int64_t)blockIdx.y * kM;
  if (m0 >= rows) return;
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5), lane = lane_id();
  if (n >= a.outputs) return;
  const int8_t* w = a.w + (int64_t)n * a.w_ld;
  const float ws = load_fresh(a.w_scale + n), b = a.bias ? load_fresh(a.bias + n) : 0.f;
  const float xs = lane < kM && m0 + lane < rows ? load_fresh(a.x_scale + m0 + lane) : 0.f;
  const int8_t* x[kM];
  int acc[kM];
#pragma unroll
  for (int m = 0; m < kM; ++m) x[m] = a.x + (m0 + m < rows ? m0 + m : rows - 1) * a.x_ld, acc[m] = 0;
  using P = Pack<int8_t, kBytes>;
  auto one = [&](const P& pw, int k) {
    P rows_of[kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) rows_of[m] = *reinterpret_cast<const P*>(x[m] + k);
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const P px = rows_of[m];
      if constexpr (kBytes == 16) {
        const int4 x4 = *reinterpret_cast<const int4*>(&px), w4 = *reinterpret_cast<const int4*>(&pw);
        acc[m] = __dp4a(x4.x, w4.x, acc[m]), acc[m] = __dp4a(x4.y, w4.y, acc[m]);
        acc[m] = __dp4a(x4.z, w4.z, acc[m]), acc[m] = __dp4a(x4.w, w4.w, acc[m]);
      } else {
        acc[m] += (int)px.v[0] * (int)pw.v[0];
      }
    }
  };
  constexpr int kAhead = 8;
  const int whole = a.inputs / kBytes * kBytes;
  int k = lane * kBytes;
  for (; k + (kAhead - 1) * 32 * kBytes < whole; k += kAhead * 32 * kBytes) {
    P pw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) pw[i] = *reinterpret_cast<const P*>(w + k + i * 32 * kBytes);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) one(pw[i], k + i * 32 * kBytes);
  }
#pragma unroll 2
  for (; k < whole; k += 32 * kBytes) one(*reinterpret_cast<const P*>(w + k), k);
  if (kBytes > 1)  // what is left of the rows
    for (k = whole + lane; k < a.inputs; k += 32)
#pragma unroll
      for (int m = 0; m < kM; ++m) acc[m] += (int)x[m][k] * (int)w[k];
  float mine = 0.f;
#pragma unroll
  for (int m = 0; m < kM; ++m) {
    const int sum = __reduce_add_sync(0xffffffffu, acc[m]);
    if (lane == m) mine = (float)sum;
  }
  if (lane < kM && m0 + lane < rows) ((T*)a.out)[(m0 + lane) * a.outputs + n] = from_f32<T>(fmaf(mine * ws, xs, b));
}

// ---- tensor cores -----------------------------------------------------------------------------------------------------
constexpr int kTileRows = 128;    // rows of a CTA
constexpr int kBlockK = 128;      // channels of the sum a stage holds: one 128-byte swizzled row
constexpr int kMaxStages = 8;
constexpr int kMaxCols = 256;     // output channels of a tile
constexpr int kMaxAcc = 8;        // accumulators in tensor memory, whose 512 columns hold two of the widest tiles
constexpr int kEpilogueSets = 4;  // of four warps, one for each quarter of an accumulator's lanes
constexpr int kEpilogueWarps = 4 * kEpilogueSets;
constexpr int kThreads = (kEpilogueWarps + 2) * 32;
constexpr int kPiece = 64;             // bytes of a row that an epilogue warp puts in order at a time
constexpr int kStaging = 32 * kPiece;  // of its 32 rows
constexpr uint32_t kABytes = kTileRows * kBlockK;

struct TcArgs {
  LinearArgs l;
  int cols;        // output channels of a tile
  int col_tiles;
  uint64_t inverse;  // of col_tiles, see Tiles
  int stages, k_blocks, accs;
  uint32_t stage_bytes;
  uint32_t idesc;
  uint32_t wait_limit;  // cycles after which a wait gives up
  int out_piece;   // bytes, 16 at most, that the output's rows start on; with 16 it has a map
};

struct Shared {
  uint64_t full[kMaxStages];   // TMA -> MMA
  uint64_t empty[kMaxStages];  // MMA -> TMA
  uint64_t acc_full[kMaxAcc];   // MMA -> epilogue
  uint64_t acc_empty[kMaxAcc];  // epilogue -> MMA
  uint64_t drained;            // MMA: all products
  uint32_t tmem;
  int abort;
  alignas(16) float scale[kEpilogueWarps][2][32];  // of a warp's piece: weight scales, bias
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of this CTA's `p` in CTA 0 of the cluster.
__device__ __forceinline__ uint32_t in_leader(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory");
}
template <int kCta> __device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  if (kCta == 1) mbar_arrive(bar);
  else asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(bar)) : "memory");
}
// A box of the tensor into this CTA's shared memory; with two CTAs to a tile its bytes count on the leader's barrier.
template <int kCta> __device__ __forceinline__ void load_box(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y) {
  if (kCta == 1)
    tma_load_2d(map, bar, dst, x, y);
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(in_leader(bar)), "r"(x), "r"(y) : "memory");
}
template <int kCta> __device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (kCta == 1)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// The barrier, in both CTAs of a pair, learns that all products issued so far are done.
template <int kCta> __device__ __forceinline__ void commit(uint64_t* bar) {
  if (kCta == 1)
    umma_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
// The same for this CTA's barrier alone.
template <int kCta> __device__ __forceinline__ void commit_here(uint64_t* bar) {
  if (kCta == 1)
    umma_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int kCta> __device__ __forceinline__ void alloc_tmem(uint32_t* dst) {
  if (kCta == 1) {
    tmem_alloc(dst, 512);
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int kCta> __device__ __forceinline__ void free_tmem(uint32_t addr) {
  if (kCta == 1) tmem_dealloc(addr, 512);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(addr) : "memory");
}
// This CTA's (pair's) tiles: first, first + step, ... below count.  Eight rows of tiles go side by side, so that what is worked
// on at a time needs as few rows and weights as can be (8192 x 4096 -> 8192: 74 tiles one row after the other need all
// weights).
struct Tiles {
  int first, step, count, row_tiles, col_tiles;
  uint64_t inverse;  // 2^40 / col_tiles, rounded up
  __device__ __forceinline__ int2 at(int t) const {  // row, column
    if (col_tiles == 1) return make_int2(t, 0);
    // t / 8 < 2^27 and fewer than 2^13 columns of tiles: the quotient is exact
    const int b = (int)(((uint64_t)(uint32_t)(t >> 3) * inverse) >> 40), r = t - b * 8 * col_tiles;
    if (8 * b + 8 <= row_tiles) return make_int2(8 * b + (r & 7), r >> 3);
    const int high = row_tiles - 8 * b;  // the last rows
    return make_int2(8 * b + r % high, r / high);
  }
};
// A box of this warp's staging to the output.
__device__ __forceinline__ void store_box(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"((uint64_t)map), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// A warp's 32 rows of staging, rows from row0 and columns from col0 on, to the output by plain stores of kBytes, which the output's
// rows are multiples of: 64 bytes of a row side by side.
template <class T, int kBytes>
__device__ __forceinline__ void store_rows(const unsigned char* mine, T* out, int outputs, int64_t row0, int64_t rows, int col0) {
  using P = Pack<T, kBytes / (int)sizeof(T)>;
  constexpr int kLanes = kPiece / kBytes, kAtOnce = 32 / kLanes;
  const int at = lane_id() % kLanes * kBytes, c = col0 + at / (int)sizeof(T);
  if (c >= outputs) return;
  int row = lane_id() / kLanes;
  out += (row0 + row) * outputs + c;
#pragma unroll(kLanes < 8 ? kLanes : 8)
  for (int i = 0; i < kLanes; ++i, row += kAtOnce, out += (int64_t)kAtOnce * outputs)
    if (row0 + row < rows)
      *reinterpret_cast<P*>(out) = *reinterpret_cast<const P*>(mine + row * kPiece + ((at >> 4) ^ (row >> 1 & 3)) * 16 + at % 16);
}
// The same for 16-bit results in pieces of 8 bytes or 4 (149 k rows 240 -> 188, two bytes / eight: 39.0 / 29.4 us; 30 k rows 128 -> 1004
// 39.6 / 25.4; of 32-bit results eight bytes were no faster than four).  Not inlined: the epilogue of whole tiles has no registers
// to spare for it (238 k rows 64 -> 192 fp16, inlined / not: 31.1 / 29.8 us).
template <class T>
__device__ __noinline__ void store_rows_in(int bytes, const unsigned char* mine, T* out, int outputs, int64_t row0, int64_t rows, int col0) {
  if (bytes == 8) store_rows<T, 8>(mine, out, outputs, row0, rows, col0);
  else store_rows<T, 4>(mine, out, outputs, row0, rows, col0);
}
// kCta CTAs share a tile of kCta * 128 rows: each holds its rows and its share of the weight rows, CTA 0 issues the products.
template <int kCta, class T>
__global__ void __launch_bounds__(kThreads, 1)
linear_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
              const __grid_constant__ CUtensorMap map_out, const TcArgs p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* staging = ring + p.stages * p.stage_bytes;
  Shared* sh = reinterpret_cast<Shared*>(staging + kEpilogueWarps * kStaging);
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const uint32_t rank = kCta == 1 ? 0 : cluster_rank();
  if (threadIdx.x == 32) prefetch_map(&map_x), prefetch_map(&map_w), prefetch_map(&map_out);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) mbar_init(&sh->full[s], 1), mbar_init(&sh->empty[s], 1);
    for (int b = 0; b < kMaxAcc; ++b) mbar_init(&sh->acc_full[b], 1), mbar_init(&sh->acc_empty[b], kCta * kEpilogueWarps);
    mbar_init(&sh->drained, 1);
    sh->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kEpilogueWarps + 1) alloc_tmem<kCta>(&sh->tmem);
  tc_fence_before();
  __syncthreads();
  if (kCta == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  volatile int* abort_flag = &sh->abort;
  pdl_release();
  pdl_wait();  // so far nothing of the kernels before has been touched
  const int64_t rows = live_rows(p.l.rows, p.l.num_rows);
  const int row_tiles = (int)((rows + kCta * kTileRows - 1) / (kCta * kTileRows));
  const Tiles tiles = {(int)(blockIdx.x / kCta), (int)(gridDim.x / kCta), row_tiles * p.col_tiles, row_tiles, p.col_tiles, p.inverse};

  if (warp == kEpilogueWarps) {
    if (lane == 0) {
      int stage = 0, phase = 0;
      bool ok = true;
      for (int t = tiles.first; ok && t < tiles.count; t += tiles.step) {
        const int2 tile = tiles.at(t);
        const int m0 = (tile.x * kCta + (int)rank) * kTileRows, n0 = tile.y * p.cols + (int)rank * (p.cols / kCta);
        for (int k = 0; k < p.k_blocks; ++k) {
          ok = mbar_wait(&sh->empty[stage], phase ^ 1, abort_flag, 1, p.wait_limit);
          if (!ok) break;
          unsigned char* a = ring + stage * p.stage_bytes;
          if (rank == 0) mbar_arrive_expect_tx(&sh->full[stage], kCta * p.stage_bytes);
          load_box<kCta>(&map_x, &sh->full[stage], a, k * kBlockK, m0);
          load_box<kCta>(&map_w, &sh->full[stage], a + kABytes, k * kBlockK, n0);
          if (++stage == p.stages) stage = 0, phase ^= 1;
        }
      }
      // The CTAs do not end with copies on their way, whoever has given up.  Those of both count on the leader's barriers; but where
      // that has given up first the other one's last ones do not, so the other one waits for the products of what it has
      // brought, or as long as no copy takes.
      mbar_drain_ring(rank == 0 ? sh->full : sh->empty, p.stages, stage, phase);
    }
  } else if (warp == kEpilogueWarps + 1) {
    // The whole warp walks by counters and one lane of it waits and issues: what feeds an MMA has to be the same for all lanes in a
    // way the compiler can see.  By a loop of one lane four products and a commit took 566 cycles where the tensor cores want
    // 512, and with the wait in front of them 840.
    if (rank == 0) {
      constexpr uint32_t kHigh = 64u | (1u << 14) | (2u << 29);  // rows in groups of eight 1024 bytes apart, 128-byte swizzle
      const uint32_t low0 = ((smem_u32(ring) & 0x3FFFFu) >> 4) | (1u << 16), low_step = p.stage_bytes >> 4;
      const int last = (p.l.inputs - (p.k_blocks - 1) * kBlockK + 31) / 32;  // products of the last stage
      int stage = 0, phase = 0, buf = 0, acc_phase = 0;
      bool bad = false;
      for (int t = tiles.first; t < tiles.count; t += tiles.step) {
        if (!bad) bad = !mbar_wait(&sh->acc_empty[buf], acc_phase ^ 1, abort_flag, 2, p.wait_limit);
        bad = __any_sync(0xffffffffu, bad);
        if (bad) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * p.cols;
        for (int k = 0; k < p.k_blocks; ++k) {
          const uint32_t low = low0 + stage * low_step;
          const uint64_t da = (uint64_t)kHigh << 32 | low, db = (uint64_t)kHigh << 32 | (low + (kABytes >> 4));
          const int n = k == p.k_blocks - 1 ? last : 4;
          if (elect_one()) {
            if (!bad) bad = !mbar_wait(&sh->full[stage], phase, abort_flag, 3, p.wait_limit);
            if (!bad) {
              tc_fence_after();
              // 32 channels further is 32 bytes further
              mma_i8<kCta>(d, da, db, p.idesc, k > 0);
              if (n > 1) mma_i8<kCta>(d, da + 2, db + 2, p.idesc, 1);
              if (n > 2) mma_i8<kCta>(d, da + 4, db + 4, p.idesc, 1);
              if (n > 3) mma_i8<kCta>(d, da + 6, db + 6, p.idesc, 1);
              commit<kCta>(&sh->empty[stage]);
              if (k == p.k_blocks - 1) commit<kCta>(&sh->acc_full[buf]);
            }
          }
          __syncwarp();
          if (++stage == p.stages) stage = 0, phase ^= 1;
        }
        if (++buf == p.accs) buf = 0, acc_phase ^= 1;
      }
      // Nor with products on their way: the epilogue may have given up on what has been issued here.
      if (elect_one()) {
        commit_here<kCta>(&sh->drained);
        mbar_drain(&sh->drained, 0);
      }
    }
  } else {
    // Four sets of four warps; a warp reads its quarter of the accumulator's lanes, the sets take turns in pieces of 64 bytes a row,
    // over the ends of tiles.  What such a piece takes is a chain of trips (tensor memory, scales, shared memory, the store), so it
    // is warps that count, and nothing that makes them wait for each other: with two sets of 128 bytes and a barrier a tile 238 k
    // rows of 64 -> 192 took 55 us.  A piece goes through shared memory, 16 bytes of row r at place j ^ (r / 2) of four, which
    // is what a tensor map with 64-byte swizzle takes out.
    constexpr int kCols = kPiece / (int)sizeof(T);  // columns of a piece
    constexpr int kVec = 16 / (int)sizeof(T);
    const int quarter = warp & 3, set = warp >> 2, pieces = p.cols / kCols;
    unsigned char* mine = staging + warp * kStaging;
    float *ws = sh->scale[warp][0], *bs = sh->scale[warp][1];
    // the warp's next piece, whose scales, a column and a row a lane, are on their way
    int next_t = tiles.first, piece = set, of_tile = -1;
    int m = 0, n_tile = 0;
    float next_w = 0.f, next_b = 0.f, next_x = 0.f;
    auto ask = [&] {
      while (piece >= pieces) piece -= pieces, next_t += tiles.step;
      if (next_t >= tiles.count) return;
      if (next_t != of_tile) {
        const int2 tile = tiles.at(next_t);
        m = (tile.x * kCta + (int)rank) * kTileRows + quarter * 32, n_tile = tile.y * p.cols, of_tile = next_t;
        next_x = m + lane < rows ? load_fresh(p.l.x_scale + m + lane) : 0.f;
      }
      const int n = n_tile + piece * kCols + lane;
      const bool in = lane < kCols && n < p.l.outputs;
      next_w = in ? load_fresh(p.l.w_scale + n) : 0.f, next_b = in && p.l.bias ? load_fresh(p.l.bias + n) : 0.f;
    };
    ask();
    int buf = 0, acc_phase = 0;
    for (int t = tiles.first; t < tiles.count; t += tiles.step) {
      const bool ok = mbar_wait(&sh->acc_full[buf], acc_phase, abort_flag, 4, p.wait_limit);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      // What the MMA warp waits for is that all have loaded, not that they are done.
      auto loaded = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_leader<kCta>(&sh->acc_empty[buf]);
      };
      if (next_t != t) loaded();
      while (next_t == t) {
        const uint32_t acc = tmem + buf * p.cols + ((uint32_t)(quarter * 32) << 16) + piece * kCols;
        uint32_t r[kCols];
#pragma unroll
        for (int h = 0; h < kCols; h += 16) tmem_ld16(acc + h, r + h);
        const int64_t row0 = m;
        const int col0 = n_tile + piece * kCols;
        const float xs = next_x;
        if (lane < kCols) ws[lane] = next_w, bs[lane] = next_b;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the piece before has left
        __syncwarp();
        piece += kEpilogueSets;
        ask();
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int h = 0; h < kCols; ++h) asm volatile("" : "+r"(r[h]));
        if (next_t != t) loaded();
#pragma unroll
        for (int j = 0; j < kPiece / 16; ++j) {
          Vec<kVec> v, w, b;
#pragma unroll
          for (int q = 0; q < kVec; q += 4) {
            *reinterpret_cast<float4*>(&w.v[q]) = *reinterpret_cast<const float4*>(ws + j * kVec + q);
            *reinterpret_cast<float4*>(&b.v[q]) = *reinterpret_cast<const float4*>(bs + j * kVec + q);
          }
#pragma unroll
          for (int e = 0; e < kVec; ++e) v.v[e] = (float)(int)r[j * kVec + e];
          v = fma(mul(v, w), all<kVec>(xs), b);
          *reinterpret_cast<Pack<T, kVec>*>(mine + lane * kPiece + ((j ^ (lane >> 1 & 3)) * 16)) = narrow<T, kVec>(v);
        }
        if (p.out_piece == 16 && row0 + 32 <= rows) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) store_box(&map_out, mine, col0, (int)row0);
        } else if (p.out_piece == 16) {
          __syncwarp();
          store_rows<T, 16>(mine, (T*)p.l.out, p.l.outputs, row0, rows, col0);
        } else if (sizeof(T) == 4 || p.out_piece == (int)sizeof(T)) {
          __syncwarp();
          store_rows<T, sizeof(T)>(mine, (T*)p.l.out, p.l.outputs, row0, rows, col0);
        } else {
          __syncwarp();
          store_rows_in(p.out_piece, mine, (T*)p.l.out, p.l.outputs, row0, rows, col0);
        }
      }
      if (++buf == p.accs) buf = 0, acc_phase ^= 1;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (kCta == 2) cluster_sync();
  if (threadIdx.x == 0 && sh->abort) atomicCAS(&g_int8_error, 0, 100 + sh->abort);
  if (warp == kEpilogueWarps + 1) free_tmem<kCta>(tmem);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------
// The weights are what is read, so they take the place of the rows: a CTA multiplies 128 of them with all of up to 32 rows.  Where
// that gives too few CTAs to ask for the weights fast enough, a cluster shares a tile's sum, each CTA some of its channels.  Then
// each adds up every so many rows' sums, which all of them have put into its shared memory; they are integers, so it does
// not matter in which order.
constexpr int kFewRows = 32;
constexpr int kMaxSplits = 4;         // CTAs of a cluster (2048 -> 2048, one row: with eight 7.8 us, four 4.7)
constexpr int kFewThreads = 6 * 32;  // four warps of the epilogue, one for the copies, one for the products

struct FewArgs {
  LinearArgs l;
  int cols;        // rows of the input, rounded up to 16
  int k_blocks, splits, stages;
  int share;       // rows whose sums a CTA of a cluster adds up: every splits-th
  uint32_t stage_bytes, tmem_cols, idesc, wait_limit;
};
struct FewShared {
  uint64_t full[kMaxStages], empty[kMaxStages], done, drained;
  uint32_t tmem;
  int abort;
  float x_scale[kFewRows];
};

template <class T>
__global__ void __launch_bounds__(kFewThreads, 1)
few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const FewArgs p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* partial = reinterpret_cast<int*>(ring + p.stages * p.stage_bytes);  // [splits][share][128]
  FewShared* sh = reinterpret_cast<FewShared*>(partial + (p.splits > 1 ? p.splits * p.share * kTileRows : 0));
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const int rank = (int)cluster_rank(), n0 = (int)(blockIdx.x / p.splits) * kTileRows;
  if (threadIdx.x == 32) prefetch_map(&map_x), prefetch_map(&map_w);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) mbar_init(&sh->full[s], 1), mbar_init(&sh->empty[s], 1);
    mbar_init(&sh->done, 1), mbar_init(&sh->drained, 1);
    sh->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) tmem_alloc(&sh->tmem, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all CTAs of the cluster run before one writes into another: each thread waits for that behind its role
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const uint32_t tmem = sh->tmem;
  volatile int* abort_flag = &sh->abort;
  pdl_release();
  pdl_wait();
  const int rows = (int)live_rows(p.l.rows, p.l.num_rows);
  // no rows: nothing is copied and nothing waited for
  const int k0 = p.k_blocks * rank / p.splits, k1 = rows > 0 ? p.k_blocks * (rank + 1) / p.splits : k0;
  const int n = n0 + warp * 32 + lane;  // of an epilogue thread
  const bool mine = warp < 4 && n < p.l.outputs;
  float ws = 0.f, b = 0.f;
  bool ok = true;

  if (warp == 4) {
    if (lane == 0) {
      int stage = 0, phase = 0;
      for (int k = k0; k < k1; ++k) {
        if (!mbar_wait(&sh->empty[stage], phase ^ 1, abort_flag, 1, p.wait_limit)) break;
        unsigned char* a = ring + stage * p.stage_bytes;
        mbar_arrive_expect_tx(&sh->full[stage], p.stage_bytes);
        tma_load_2d(&map_w, &sh->full[stage], a, k * kBlockK, n0);
        tma_load_2d(&map_x, &sh->full[stage], a + kABytes, k * kBlockK, 0);
        if (++stage == p.stages) stage = 0, phase ^= 1;
      }
      mbar_drain_ring(sh->full, p.stages, stage, phase);
    }
  } else if (warp == 5) {
    constexpr uint32_t kHigh = 64u | (1u << 14) | (2u << 29);
    const uint32_t low0 = ((smem_u32(ring) & 0x3FFFFu) >> 4) | (1u << 16), low_step = p.stage_bytes >> 4;
    const int last = (p.l.inputs - (p.k_blocks - 1) * kBlockK + 31) / 32;
    int stage = 0, phase = 0;
    bool bad = false;
    for (int k = k0; k < k1; ++k) {
      const uint32_t low = low0 + stage * low_step;
      const uint64_t da = (uint64_t)kHigh << 32 | low, db = (uint64_t)kHigh << 32 | (low + (kABytes >> 4));
      const int steps = k == p.k_blocks - 1 ? last : 4;
      if (elect_one()) {
        if (!bad) bad = !mbar_wait(&sh->full[stage], phase, abort_flag, 3, p.wait_limit);
        if (!bad) {
          tc_fence_after();
          mma_i8<1>(tmem, da, db, p.idesc, k > k0);
          if (steps > 1) mma_i8<1>(tmem, da + 2, db + 2, p.idesc, 1);
          if (steps > 2) mma_i8<1>(tmem, da + 4, db + 4, p.idesc, 1);
          if (steps > 3) mma_i8<1>(tmem, da + 6, db + 6, p.idesc, 1);
          umma_commit(&sh->empty[stage]);
          if (k == k1 - 1) umma_commit(&sh->done);
        }
      }
      __syncwarp();
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
    // products are seen out as above, also where it is the epilogue that has given up on them
    if (elect_one()) {
      umma_commit(&sh->drained);
      mbar_drain(&sh->drained, 0);
    }
  } else {
    if (mine) ws = load_fresh(p.l.w_scale + n), b = p.l.bias ? load_fresh(p.l.bias + n) : 0.f;
    if ((int)threadIdx.x < rows) sh->x_scale[threadIdx.x] = load_fresh(p.l.x_scale + threadIdx.x);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (k1 > k0) ok = __all_sync(0xffffffffu, mbar_wait(&sh->done, 0, abort_flag, 4, p.wait_limit));
    tc_fence_after();
    __syncwarp();
    if (p.splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    int owner = 0, place = 0;  // of row c + e
    for (int c = 0; c < rows && ok; c += 16) {
      uint32_t r[16];
      tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, r);
      tmem_ld_wait(r);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (p.splits > 1) {
          const int* at = partial + (rank * p.share + place) * kTileRows + threadIdx.x;
          if (c + e < rows)
            asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.u32 [a], %2;\n\t}"
                         ::"r"(smem_u32(at)), "r"(owner), "r"(r[e]) : "memory");
          if (++owner == p.splits) owner = 0, ++place;
        } else if (c + e < rows && mine) {
          ((T*)p.l.out)[(int64_t)(c + e) * p.l.outputs + n] = from_f32<T>(fmaf((float)(int)r[e] * ws, sh->x_scale[c + e], b));
        }
      }
    }
  }
  __syncwarp();
  if (warp >= 4 && p.splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (p.splits > 1) cluster_sync();
  if (p.splits > 1 && warp < 4 && mine && ok) {
#pragma unroll 4
    for (int i = 0; i < p.share; ++i) {
      const int m = i * p.splits + rank;
      if (m >= rows) break;
      int sum = 0;
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
        if (s < p.splits) sum += partial[(s * p.share + i) * kTileRows + threadIdx.x];
      ((T*)p.l.out)[(int64_t)m * p.l.outputs + n] = from_f32<T>(fmaf((float)sum * ws, sh->x_scale[m], b));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && sh->abort) atomicCAS(&g_int8_error, 0, 200 + sh->abort);
  if (warp == 5) tmem_dealloc(tmem, p.tmem_cols);
}

// Rows of bytes that do not start on 16 bytes: copied so that they do.
__global__ void __launch_bounds__(256)
repitch_kernel(const int8_t* from, int64_t from_ld, int8_t* to, int64_t to_ld, int64_t rows, int channels,
               const int32_t* num_rows) {
  pdl_release();
  pdl_wait();
  rows = live_rows(rows, num_rows);
  const int words = (int)(to_ld / 4);
  const int64_t n = rows * words, nth = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += nth) {
    const int64_t row = i / words;
    const int c = (int)(i - row * words) * 4;
    const int8_t* s = from + row * from_ld + c;
    char4 v;
    v.x = c < channels ? s[0] : 0, v.y = c + 1 < channels ? s[1] : 0, v.z = c + 2 < channels ? s[2] : 0, v.w = c + 3 < channels ? s[3] : 0;
    *reinterpret_cast<char4*>(to + row * to_ld + c) = v;
  }
}

constexpr int kMaxInputs = 65536, kMaxOutputs = 65536;

bool aligned_rows(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 16 == 0; }

// Map over rows `pitch` bytes apart; boxes of box_bytes (64 or 128) by box_rows, swizzled.
bool make_map(CUtensorMap* map, CUtensorMapDataType type, int esize, const void* base, uint64_t cols, uint64_t rows, uint64_t pitch,
              uint32_t box_bytes, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch};
  cuuint32_t box[2] = {box_bytes / esize, box_rows}, elem[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            box_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Raises the kernel's limit of shared memory to all there is, once per device.
template <class K> int allow_smem(K kernel, std::mutex& lock, bool (&set)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return D3D_ERR_CUDA;
  std::lock_guard<std::mutex> guard(lock);
  if (!set[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return D3D_ERR_CUDA;
    set[dev] = true;
  }
  return D3D_OK;
}

// As a programmatic dependent of the kernel before: setting up barriers and tensor memory and fetching the maps takes 2 us, which
// can be beside its end.
template <class K, class... A> int launch_cluster(K kernel, int ctas, int cluster, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? D3D_OK : D3D_ERR_CUDA;
}

template <class T> int launch_dot(const LinearArgs& a, cudaStream_t st) {
  const bool wide = aligned_rows(a.x, a.x_ld) && aligned_rows(a.w, a.w_ld);
  const unsigned gx = (unsigned)ceil_div(a.outputs, 8);
#define D3D_DOT(M)                                                         \
  do {                                                                     \
    const dim3 grid(gx, (unsigned)ceil_div(a.rows, M));                    \
    D3D_LAUNCH(true, (wide ? dot_kernel<T, M, 16> : dot_kernel<T, M, 1>), grid, 256, 0, st, a); \
  } while (0)
  if (a.rows == 1) D3D_DOT(1);
  else if (a.rows == 2) D3D_DOT(2);
  else if (a.rows <= 4) D3D_DOT(4);
  else D3D_DOT(8);
#undef D3D_DOT
  return D3D_OK;
}

template <class T> int launch_few(const LinearArgs& a, cudaStream_t st) {
  FewArgs p;
  p.l = a;
  p.cols = (int)align_up(a.rows, 16);
  p.k_blocks = (int)ceil_div(a.inputs, kBlockK);
  const int tiles = (int)ceil_div(a.outputs, kTileRows);
  p.splits = kNumSMs / tiles;
  if (p.splits > kMaxSplits) p.splits = kMaxSplits;
  if (p.splits > p.k_blocks / 2) p.splits = p.k_blocks / 2;
  if (p.splits < 1) p.splits = 1;
  p.share = (int)ceil_div(a.rows, p.splits);
  p.stage_bytes = kABytes + (uint32_t)p.cols * kBlockK;
  const size_t fixed = 1024 + (p.splits > 1 ? (size_t)p.splits * p.share * kTileRows * 4 : 0) + sizeof(FewShared);
  p.stages = (int)((227 * 1024 - fixed) / p.stage_bytes);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.tmem_cols = 32;
  p.wait_limit = wait_limit();
  p.idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.cols >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
  CUtensorMap map_w, map_x;
  if (!make_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, a.inputs, a.outputs, a.w_ld, kBlockK, kTileRows) ||
      !make_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.x, a.inputs, a.rows, a.x_ld, kBlockK, p.cols))
    return D3D_ERR_CUDA;
  static std::mutex lock;
  static bool set[64] = {};
  const int rc = allow_smem(few_rows_kernel<T>, lock, set);
  if (rc != D3D_OK) return rc;
  return launch_cluster(few_rows_kernel<T>, tiles * p.splits, p.splits, kFewThreads, fixed + p.stages * p.stage_bytes, st, map_w, map_x, p);
}

template <int kCta, class T> int launch_tiles(const LinearArgs& a, int cols, cudaStream_t st) {
  TcArgs p;
  p.l = a;
  p.cols = cols;
  p.col_tiles = (int)ceil_div(a.outputs, cols);
  p.inverse = ((1ull << 40) + p.col_tiles - 1) / p.col_tiles;
  p.k_blocks = (int)ceil_div(a.inputs, kBlockK);
  p.accs = 512 / cols < kMaxAcc ? 512 / cols : kMaxAcc;
  p.stage_bytes = kABytes + (uint32_t)(cols / kCta) * kBlockK;
  const size_t fixed = 1024 + kEpilogueWarps * kStaging + sizeof(Shared);
  p.stages = (int)((227 * 1024 - fixed) / p.stage_bytes);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  // D 32-bit integers, A and B signed
  p.idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(kCta * kTileRows >> 4) << 24);
  p.wait_limit = wait_limit();
  p.out_piece = 16;
  while ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)a.outputs * sizeof(T)) % p.out_piece) p.out_piece /= 2;
  CUtensorMap map_x, map_w, map_out = {};
  constexpr CUtensorMapDataType kType = sizeof(T) == 4                        ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                        : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!make_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.x, a.inputs, a.rows, a.x_ld, kBlockK, kTileRows) ||
      !make_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, a.inputs, a.outputs, a.w_ld, kBlockK, cols / kCta) ||
      (p.out_piece == 16 && !make_map(&map_out, kType, sizeof(T), a.out, a.outputs, a.rows, a.outputs * sizeof(T), kPiece, 32)))
    return D3D_ERR_CUDA;
  static std::mutex lock;
  static bool set[64] = {};
  const int rc = allow_smem(linear_kernel<kCta, T>, lock, set);
  if (rc != D3D_OK) return rc;
  const int64_t tiles = ceil_div(a.rows, kCta * kTileRows) * p.col_tiles;
  return launch_cluster(linear_kernel<kCta, T>, (int)(kCta * (tiles < kNumSMs / kCta ? tiles : kNumSMs / kCta)), kCta, kThreads,
                        fixed + p.stages * p.stage_bytes, st, map_x, map_w, map_out, p);
}

// Output channels of a tile, a multiple of `unit`: such that the rounds of tiles over `units` CTAs (or pairs) take least.  A round
// lasts as its tile's channels and what does not depend on them, the rows that come in and the hand-overs, about 96 of them (us,
// as few tiles as fill the GPU / this: 14 k rows 752 -> 592 17.0 / 15.5, 3000 rows 768 -> 2304 10.3 / 8.8, 5000 rows 2048 -> 2048
// in 32 bits 23.6 / 21.0; 66 k rows 256 -> 512, where both are the same tiles, 19.4).
int tile_cols(int64_t row_tiles, int outputs, int unit, int units) {
  int best = unit;
  int64_t least = INT64_MAX;
  for (int cols = unit; cols <= kMaxCols; cols += unit) {
    const int64_t n = ceil_div(outputs, cols), cost = ceil_div(row_tiles * n, units) * (cols + 96);
    if (cost <= least && (cols == unit || ceil_div(outputs, cols - unit) > n)) least = cost, best = cols;
  }
  return best;
}

// Two CTAs to a tile, which halves what the weights cost, for long sums over enough tiles; short ones are bound by the epilogue,
// where a pair waits for the slower one.  us with one / two: 66 k rows, 512 outputs, 512 inputs 26.8 / 34.1, 1024 39.0 / 39.5,
// 2048 65.9 / 57.2; 16 k rows, 1024 outputs, 1024 inputs 21.0 / 22.7, 2048 32.9 / 30.9; 8192 x 4096 -> 8192 207 / 178.
// The products want multiples of 16 channels, of 32 with two CTAs, and the output leaves in pieces of 64 bytes a row, which tiles
// consist of.
template <class T> int launch_linear(const LinearArgs& a, cudaStream_t st) {
  constexpr int kCols = kPiece / (int)sizeof(T);
  const int64_t pairs = ceil_div(a.rows, 2 * kTileRows) * ceil_div(a.outputs, kMaxCols);
  if (pairs >= kNumSMs / 2 && a.inputs > 1024)
    return launch_tiles<2, T>(a, tile_cols(ceil_div(a.rows, 2 * kTileRows), a.outputs, 32, kNumSMs / 2), st);
  return launch_tiles<1, T>(a, tile_cols(ceil_div(a.rows, kTileRows), a.outputs, kCols, kNumSMs), st);
}

// Whether the integer units' dot products are taken: where there is so little to multiply that setting up the tensor cores takes
// longer (us, dot products / tensor cores, launched on their own: one row 256 -> 512 4.1 / 6.3, 1024 -> 1024 4.2 / 6.3; behind
// other kernels, where the setting up is hidden, they are equal up to 2048 -> 2048, 5.4 / 4.7, and at 4096 -> 4096 8.2 / 5.6),
// and for few rows by weights that do not start on 16 bytes, where a copy of all weights to better places takes longer (dot products
// / copy and tensor cores, 1001 -> 5000, one row, four, six: 6.5 / 12.5, 10.6 / 16.5, 14.7 / 16.6; 3802 -> 3731: 12.6 / 18.9,
// 21.5 / 22.8, 33.1 / 22.9).  Where only the rows do not, the dot products read the weights by bytes too, and it is the rows that the
// others copy: twice as much work and short sums are still little (one row 512 -> 16000 4.9 / 7.2, 1008 -> 8000 6.8 / 7.2,
// 1024 -> 16384 8.2 / 7.4, 2048 -> 3584 8.8 / 7.2, 4096 -> 4096 13.2 / 7.5, four rows 33 / 7.5).
bool little(int64_t rows, int64_t inputs, int64_t outputs, bool aligned_rows, bool aligned_weights) {
  const int64_t work = rows * inputs * outputs;
  if (rows <= 64 && work <= (1 << 22)) return true;
  return aligned_weights ? !aligned_rows && rows * inputs <= 1024 && work <= (1 << 23) : rows <= 4;
}

size_t repitched(const void* p, int64_t ld, int64_t rows, int channels) {
  return aligned_rows(p, ld) ? 0 : align_up((size_t)rows * align_up(channels, 16), 256);
}

}  // namespace

int take_int8_linear_error(int* code) {
  const int zero = 0;
  if (cudaMemcpyFromSymbol(code, g_int8_error, sizeof(int)) != cudaSuccess) return D3D_ERR_CUDA;
  if (cudaMemcpyToSymbol(g_int8_error, &zero, sizeof(int)) != cudaSuccess) return D3D_ERR_CUDA;
  return D3D_OK;
}

}  // namespace d3d

using namespace d3d;

extern "C" size_t d3d_int8_linear_workspace(const int8_t* x, int64_t x_ld, int64_t rows, const int8_t* weight, int64_t weight_ld,
                                            int inputs, int outputs) {
  if (inputs < 1 || outputs < 1 || little(rows, inputs, outputs, aligned_rows(x, x_ld), aligned_rows(weight, weight_ld))) return 0;
  return repitched(x, x_ld, rows, inputs) + repitched(weight, weight_ld, outputs, inputs);
}

extern "C" int d3d_int8_linear(int dtype, const int8_t* x, int64_t x_ld, const float* x_scales, int64_t rows, const int32_t* num_rows,
                               const int8_t* weight, int64_t weight_ld, const float* weight_scales, const float* bias, int inputs,
                               int outputs, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  D3D_NVTX_RANGE("d3d_int8_linear");
  const int esize = (int)dtype_size(dtype);
  D3D_REQUIRE(dtype == D3D_FLOAT || dtype == D3D_HALF || dtype == D3D_BF16, D3D_ERR_UNSUPPORTED_DTYPE);
  D3D_REQUIRE(rows >= 0 && inputs >= 1 && outputs >= 1 && x_ld >= inputs && weight_ld >= inputs, D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(inputs <= kMaxInputs && outputs <= kMaxOutputs && rows <= (1ll << 31) - 1024 &&
                  ceil_div(rows, kTileRows) * ceil_div(outputs, 16) < (1ll << 30),
              D3D_ERR_TOO_LARGE);
  if (rows == 0) return D3D_OK;
  D3D_REQUIRE(x && x_scales && weight && weight_scales && out && on_multiples(esize, out) &&
                  on_multiples(4, x_scales, num_rows, weight_scales, bias),
              D3D_ERR_INVALID_ARGUMENT);
  const size_t need = d3d_int8_linear_workspace(x, x_ld, rows, weight, weight_ld, inputs, outputs);
  D3D_REQUIRE(need == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 256 == 0), D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace_bytes >= need, D3D_ERR_WORKSPACE_TOO_SMALL);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  LinearArgs a = {x, weight, x_ld, weight_ld, x_scales, weight_scales, bias, out, rows, num_rows, inputs, outputs};
  const bool dot = little(rows, inputs, outputs, aligned_rows(x, x_ld), aligned_rows(weight, weight_ld));
  if (!dot) {
    uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
    const int64_t pitch = (int64_t)align_up(inputs, 16);
    if (!aligned_rows(x, x_ld)) {
      D3D_LAUNCH(true, repitch_kernel, (unsigned)stream_grid(rows * (pitch / 4), 256), 256, 0, st, x, x_ld, (int8_t*)ws, pitch, rows, inputs,
                 num_rows);
      a.x = (const int8_t*)ws, a.x_ld = pitch;
      ws += repitched(x, x_ld, rows, inputs);
    }
    if (!aligned_rows(weight, weight_ld)) {
      D3D_LAUNCH(true, repitch_kernel, (unsigned)stream_grid(outputs * (pitch / 4), 256), 256, 0, st, weight, weight_ld, (int8_t*)ws, pitch,
                 (int64_t)outputs, inputs, (const int32_t*)nullptr);
      a.w = (const int8_t*)ws, a.w_ld = pitch;
    }
  }
  auto launch = [&](auto t) -> int {
    using T = decltype(t);
    if (dot) return launch_dot<T>(a, st);
    return rows <= kFewRows ? launch_few<T>(a, st) : launch_linear<T>(a, st);
  };
  switch (dtype) {
    case D3D_FLOAT: return launch(float());
    case D3D_HALF: return launch(__half());
    default: return launch(__nv_bfloat16());
  }
}
