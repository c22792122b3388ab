// The matrix products of ops/ffn.py and ops/adapters.py on tcgen05: one persistent kernel over CTA pairs.
//
//   kGated    h[M,F]  = a(x Wg^T) * (x Wu^T)     both operands K-major; a tile is 256 rows x 128 columns of h, its accumulator
//                                                holds the 128 gate columns and the 128 up columns side by side
//   kInput    dx[M,K] = dpre[M,2F] W[2F,K]       B is stored along N (MN-major)
//   kWeight   dW[2F,K] = dpre[M,2F]^T x[M,K]     both operands are stored along their outer index (MN-major)
//   kAdapt    y[M,N]  = x W^T + V_a B_a^T        both K-major; behind the K blocks of a tile come blocks of the low-rank factors
//                                                (see "Adapters" below)
//
// The two CTAs of a cluster share one 256 x 256 accumulator tile (cta_group::2): each loads its own 128 rows of A and 128 of the
// 256 columns of B, 32 KB a K block of 64, into a six-stage ring; the even CTA issues the MMAs for both.  For kGated the first
// CTA's half of B are the gate rows of W and the second's the up rows, so gate and up of one h are 128 TMEM columns apart in the
// same lane, and the product with the activation never leaves the thread.
//   warp 0      TMA producer
//   warp 1      MMA issuer (even CTA), owns the 512 TMEM columns: two accumulators, so a tile's epilogue runs under the next
//               tile's main loop
//   warps 2-9   epilogue, two per TMEM lane quarter with half of the columns each: tcgen05.ld, activation, BF16, a 32 x 64 slab per
//               warp in swizzled shared memory, TMA store
//   warps 10-11 kAdapt: the blocks of low-rank factors
// Bound by the tensor pipe under the power cap: forward 4096 x 8192, K = 6144: 632 us, 1305 TFLOP/s, where a library product of these
// sizes without the activation takes 568 - 611; 2048 x 2048, K = 6144: 70 - 73 us (82).  At 4096 x 2048 the pipe is busy for 76 (forward), 82
// (dx) and 82 % (dW) of the kernel, at 1.54 GHz; a K block takes a pair 0.31 us, about 8 us go to launch, the first loads, the
// last tile's epilogue and the end.  Calls of one or two waves of tiles leave units idle (1031 x 1368: 55 tiles for 74 units, 42 us).
// Ragged sizes need no code in the main loop: tensor maps fill with zeros beyond their extents and stores are clipped.
//
// MN-major tiles: a box of 64 (outer index, 128 bytes, swizzled) x 64 K rows is 8 KB; a tile of 128 is two boxes.  In the
// descriptor the leading offset is the distance between boxes (8192), the stride offset that between groups of 8 K rows (1024).
#pragma once
#include <atomic>
#include <cstring>
#include <optional>
#include <cuda_bf16.h>
#include "../include/fp4ar_layer.h"
#include "../include/fp4ar_tensor.cuh"
#include "activation.cuh"
#include "host_util.h"
#include "split_space.h"
#include "tensor_map.h"

namespace fp4ar {
namespace layer {

enum : int { kGated = 0, kInput = 1, kWeight = 2, kAdapt = 3 };

constexpr int kRowsCta = 128, kBlockK = 64, kStages = 6;
template <int OP> constexpr int kThreads = OP == kAdapt ? 384 : 320;
constexpr int kOpBytes = kRowsCta * kBlockK * 2;               // 16 KB of A, 16 KB of B per CTA and stage
constexpr int kStage = 2 * kOpBytes;
constexpr int kSlab = 32 * 64 * 2;                             // 32 rows x 64 BF16 columns, one warp's store
constexpr int kSlabs = 8 * kSlab;                              // one per epilogue warp
constexpr int kSmemBytes = kStages * kStage + kSlabs + 768 + 1024;
constexpr int kListStride = 260;                               // per 256-row tile: count, then up to 256 adapters (16-byte pitch)
constexpr int kVerdicts = 16;                                  // a granted stage is six segments ahead of the MMAs at most, these two of the epilogue
constexpr int kChunk = 32;                                     // ranks per block of low-rank factors

struct Params {
  int M, N;                 // rows and columns of the output (kGated: columns of h)
  int kblocks;
  int act;
  bool want_pre;
  int cut_units;            // units that share the cut tiles, 0: none are cut (see Walk)
  float* partial;           // [CTA][8][8][128] float4
  uint32_t* flags;          // [CTA][kSplitFlags]: 1 = that epilogue warp's part of the slot is written and not yet consumed
  // adapters
  int R, adapters;
  const int* ids;           // [M]
  const __nv_bfloat16* v;   // [M][chunks of 32 ranks][64] scaled x A^T: the rounded values, then what the rounding left
  const int* lists;         // [row tiles][kListStride]
  const __nv_bfloat16* b;   // [adapters][N][R]
  StatusWords* status;
  unsigned long long timeout_ns;
};
struct Maps { CUtensorMap a, b, out, pre, low; };              // `pre`: kGated; `low`: B of the adapters

// Descriptor of an MN-major tile (see above).
__device__ __forceinline__ uint64_t umma_desc_mn128(const void* smem_tile) {
  uint64_t d = (uint64_t)((smem_addr(smem_tile) >> 4) & 0x3FFFu);
  d |= (uint64_t)(8192 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ bool mbar_test_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{ .reg .pred p;\n"
               "  mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
               "  selp.u32 %0, 1, 0, p; }"
               : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
  return done != 0;
}
// Without release: what the arrival says (this warp's TMEM loads are through) needs no memory of the thread to be written first, and
// waiting for that took 1.6 us at the end of every tile.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// Nobody of the cluster goes on before all are here; orders no memory.
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, const void* smem_src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(smem_addr(smem_src))
               : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int x, int y, int z, const void* smem_src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y),
               "r"(z), "r"(smem_addr(smem_src))
               : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Tiles in panels of 8 columns of tiles, as the NVFP4 GEMM walks them: the tiles in flight share operands in L2.
constexpr int kPanelTiles = 8;
__host__ __device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int& m, int& n) {
  const int per_panel = m_tiles * kPanelTiles;
  const int panel = t / per_panel, within = t - panel * per_panel;
  const int left = n_tiles - panel * kPanelTiles, width = left < kPanelTiles ? left : kPanelTiles;
  m = within / width;
  n = panel * kPanelTiles + within % width;
}

// The work of a unit (CTA pair) as a list of segments (tile, K blocks [lo, lo + count)), the same list in all roles.
//   whole tiles:  unit, unit + units, ...
//   cut tiles:    where the tiles do not fill the units evenly, the first `cut` of them (units + remainder, or all of them where there
//                 are fewer tiles than units) are laid out as tiles x kblocks blocks and cut into cut_units equal ranges.
//                 Where the boundary of two ranges falls into a tile, the unit whose range ENDS there finishes the tile: it runs
//                 the tile's LAST K blocks and adds what the units behind it (one, or several where a range is shorter than a
//                 tile) leave in their slots.  A range that begins inside a tile runs that share first, so nobody waits for
//                 work that waits for him, and every unit leaves one partial at most.  Sums are taken in the order of the units.
enum : int { kWhole = 0, kProduce = 1, kFinish = 2 };
struct Seg { int tile, lo, count, kind, others; };       // others: of kFinish, units behind this one that share the tile
struct Walk {
  int tiles, kblocks, units, cut_units, unit, t;
  long long total, u, end;
  __host__ __device__ Walk(int tiles_, int kblocks_, int unit_, int units_, int cut_units_)
      : tiles(tiles_), kblocks(kblocks_), units(units_), cut_units(cut_units_), unit(unit_) {
    const int cut = cut_units ? (tiles < units ? tiles : units + tiles % units) : 0;
    total = (long long)cut * kblocks;
    u = unit < cut_units ? total * unit / cut_units : 0;
    end = unit < cut_units ? total * (unit + 1) / cut_units : 0;
    t = cut + unit;
  }
  __host__ __device__ bool next(Seg& s) {
    if (u < end) {
      s.tile = (int)(u / kblocks);
      const long long at = (long long)s.tile * kblocks;
      const int off = (int)(u - at);
      s.count = (int)(end - u < kblocks - off ? end - u : kblocks - off);
      s.others = 0;
      if (off > 0) {
        int f = unit - 1;                              // the finisher: its range holds the tile's first block
        while (total * f / cut_units > at) f--;
        s.kind = kProduce;
        s.lo = off - (int)(total * (f + 1) / cut_units - at);
      } else if (s.count < kblocks) {
        s.kind = kFinish;
        s.lo = kblocks - s.count;
        for (int f = unit + 1; total * f / cut_units < at + kblocks; f++) s.others++;
      } else {
        s.kind = kWhole;
        s.lo = 0;
      }
      u += s.count;
      return true;
    }
    if (t >= tiles) return false;
    s.tile = t; s.lo = 0; s.count = kblocks; s.kind = kWhole; s.others = 0;
    t += units;
    return true;
  }
};

// ---- Adapters.  y_i = x_i W^T + sum_r V[i][r] B_a[:, r], a = ids[i].  A 256-row tile has a list of the adapters its rows use; for
// each of them and every 32 ranks follows one more block of the same accumulation: A is V of the rows that have this adapter and
// zero elsewhere, as two BF16 halves (columns 0-31 the rounded value, 32-63 what the rounding left, so V counts with 16 bits), B is
// B_a [128 columns x ranks], used twice.  Two warps of their own fill the A blocks, while the producer goes on with the K blocks of
// the next tile: one warp that did both took 5 us a block.
// 0 x infinity would leak one request's broken adapter into the rows of others: those warps look through the 256 rows of B_a that a
// tile takes (they come from L2, under the main loop) and write zeros for A and B where one value is not finite; the
// epilogue then adds such adapters to their own rows by plain dot products.
constexpr int kLowThreads = 64, kLowAhead = 3;      // (fewer than the ring's stages: a grant needs the blocks six before it handed over)
// 16 bytes into shared memory without a register in between, or zeros
__device__ __forceinline__ void copy_or_zero(void* smem_dst, const void* gmem_src, bool copy) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(smem_dst)), "l"(gmem_src), "r"(copy ? 16 : 0) : "memory");
}
__device__ __forceinline__ void low_rank_barrier() { asm volatile("barrier.cta.sync 1, 64;" ::: "memory"); }
// ... and whether every one of the two warps' threads says yes
__device__ __forceinline__ bool low_rank_all(bool yes) {
  uint32_t v = yes;
  asm volatile("{ .reg .pred p, r;\n"
               "  setp.ne.u32 p, %0, 0;\n"
               "  barrier.cta.red.and.pred r, 1, 64, p;\n"
               "  selp.u32 %0, 1, 0, r; }"
               : "+r"(v)::"memory");
  return v != 0;
}

// Not zero where one of two BF16 values is infinite or NaN (all eight exponent bits set).
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }
// Rows n0 .. n0 + 255 (below N) of B of one adapter: are all values finite?  By a warp (every lane has the answer) or by one thread.
template <int LANES>
__device__ __forceinline__ bool low_rank_finite(const Params& p, int adapter, int n0, int lane) {
  const uint4* b = reinterpret_cast<const uint4*>(p.b + ((size_t)adapter * p.N + n0) * p.R);
  const int n = min(256, p.N - n0) * (p.R / 8);
  uint32_t bad = 0;
  for (int i = lane; i < n; i += 16 * LANES) {               // sixteen loads in flight
    uint4 w[16];
#pragma unroll
    for (int j = 0; j < 16; j++) w[j] = __ldg(b + min(i + j * LANES, n - 1));
#pragma unroll
    for (int j = 0; j < 16; j++) bad |= not_finite(w[j].x) | not_finite(w[j].y) | not_finite(w[j].z) | not_finite(w[j].w);
  }
  return LANES == 1 ? bad == 0 : (bool)__all_sync(0xffffffffu, bad == 0);
}
static __device__ __noinline__ bool low_rank_unsafe(const Params& p, int adapter, int n0) { return !low_rank_finite<1>(p, adapter, n0, 0); }

static __device__ __noinline__ float low_rank_dot(const __nv_bfloat16* v, const __nv_bfloat16* b, int R) {
  float s = 0.0f;
  for (int r = 0; r < R; r++) {
    const unsigned short* line = reinterpret_cast<const unsigned short*>(v) + (r / kChunk) * 64 + r % kChunk;
    s = fmaf(bf16_lo(__ldcg(line)) + bf16_lo(__ldcg(line + 32)), __bfloat162float(b[r]), s);
  }
  return s;
}

template <int OP>
__global__ void __launch_bounds__(kThreads<OP>, 1)
pair_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  constexpr bool kAMn = OP == kWeight, kBMn = OP == kWeight || OP == kInput;
  constexpr int kTileN = OP == kGated ? 128 : 256;             // output columns per tile
  constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((kAMn ? 1u : 0u) << 15) | ((kBMn ? 1u : 0u) << 16) |
                              ((256u >> 3) << 17) | ((256u >> 4) << 24);       // F32 += BF16 x BF16, N = 256, M = 256
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* slabs = ring + kStages * kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(slabs + kSlabs);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* settled = acc_empty + 2;
  uint64_t* granted = settled + 1;             // kAdapt, [kStages]: the stage is free for a block of low-rank factors
  uint64_t* filled = granted + kStages;        // kAdapt, [kStages], second CTA: its half of such a block is written
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(filled + kStages);
  volatile uint32_t* abort_flag = tmem_holder + 1;
  volatile uint32_t* unsafe_tile = tmem_holder + 2;            // kAdapt, [kVerdicts]: 1 + the segment of which an adapter is left to the epilogue
  uint8_t* skipped = reinterpret_cast<uint8_t*>(tmem_holder + 2 + kVerdicts);      // kAdapt, [256]: this tile's adapters that are left to the epilogue
  uint32_t issued = 0;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m_tiles = (p.M + 255) / 256, n_tiles = (p.N + kTileN - 1) / kTileN, tiles = m_tiles * n_tiles;
  const uint32_t crank = cluster_cta_rank();
  const bool leads = crank == 0u;
  Walk walk(tiles, p.kblocks, blockIdx.x / 2, gridDim.x / 2, p.cut_units);
  Seg sg;

  if (threadIdx.x == 0) {
    // kAdapt: two arrivals, since both CTAs write into a stage of low-rank factors themselves
    for (int s = 0; s < kStages; s++) { mbar_init(full + s, OP == kAdapt ? 2 : 1); mbar_init(empty + s, 1); mbar_init(granted + s, 1); mbar_init(filled + s, 1); }
    for (int a = 0; a < 2; a++) { mbar_init(acc_full + a, 1); mbar_init(acc_empty + a, 16); }
    mbar_init(settled, 1);
    *abort_flag = 0u;
    for (int i = 0; i < kVerdicts; i++) unsafe_tile[i] = 0u;
    mbar_init_fence();
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
    prefetch_tensormap(&maps.out);
  }
  if (warp == 1) { tmem_alloc_pair(tmem_holder, 512); tmem_relinquish_pair(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  GemmWait gw{abort_flag, p.status, p.timeout_ns};

  // kAdapt: the launch before this one lets it start only after its own wait, so everything before that one is complete here; what that
  // one itself writes (V, the lists) is waited for by those who read it, behind the K loop of their first tile.  Not where tiles are cut:
  // another thread may have put a launch with the same slots in between, and that one has to be through.
  if (OP != kAdapt || p.cut_units) pdl_wait_prior_grids();
  pdl_release_dependents();
  auto factors_ready = [&]() { if (OP == kAdapt) pdl_wait_prior_grids(); };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      while (walk.next(sg)) {
        int tm, tn;
        tile_at(sg.tile, m_tiles, n_tiles, tm, tn);
        const int m0 = tm * 256 + (int)crank * 128;
        const int n0 = OP == kGated ? tn * 128 + (int)crank * p.N : tn * 256 + (int)crank * 128;
        for (int kb = sg.lo; kb < sg.lo + sg.count; kb++, issued++) {
          const int s = issued % kStages;
          if (!gemm_wait(empty + s, ((issued / kStages) & 1u) ^ 1u, gw, 1)) goto done;
          uint8_t *sa = ring + s * kStage, *sb = sa + kOpBytes;
          const uint32_t lead_full = cluster_addr(full + s, 0u);
          if (leads) {
            mbar_arrive_expect(full + s, 2 * kStage);
            // (the second arrival is the other CTA's for a block of low-rank factors alone: one at cluster scope for every K
            // block, and a wait at that scope, cost 90 us of 165 at M = 4096, K = 2048)
            if (OP == kAdapt) mbar_arrive(full + s);
          }
          const int k0 = kb * kBlockK;
          if constexpr (kAMn) {
            tma_load_2d_pair(sa, &maps.a, m0, k0, lead_full);
            tma_load_2d_pair(sa + 8192, &maps.a, m0 + 64, k0, lead_full);
          } else {
            tma_load_2d_pair(sa, &maps.a, k0, m0, lead_full);
          }
          if constexpr (kBMn) {
            tma_load_2d_pair(sb, &maps.b, n0, k0, lead_full);
            tma_load_2d_pair(sb + 8192, &maps.b, n0 + 64, k0, lead_full);
          } else {
            tma_load_2d_pair(sb, &maps.b, k0, n0, lead_full);
          }
        }
        if (OP == kAdapt && sg.kind != kProduce) {
          factors_ready();
          // hand the next stages, as they come free, to the warps that fill them.  (Those cannot wait for `empty` themselves: a parity
          // says nothing to who has not seen every round of a stage.)
          const int blocks = p.lists[(size_t)tm * kListStride] * ((p.R + kChunk - 1) / kChunk);
          for (int i = 0; i < blocks; i++, issued++) {
            const int s = issued % kStages;
            if (!gemm_wait(empty + s, ((issued / kStages) & 1u) ^ 1u, gw, 1)) goto done;
            mbar_arrive(granted + s);
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && leads) {
      uint32_t it = 0, tile_i = 0;
      for (; walk.next(sg); tile_i++) {
        const uint32_t a = tile_i & 1u;
        if (!gemm_wait(acc_empty + a, ((tile_i >> 1) & 1u) ^ 1u, gw, 2)) goto done;
        tc_fence_after();
        const uint32_t d = tmem_base + a * 256;
        for (int j = 0; j < sg.count; j++, it++) {
          const int s = it % kStages;
          if (!gemm_wait(full + s, (it / kStages) & 1u, gw, 3)) goto done;
          tc_fence_after();
          const uint8_t* sa = ring + s * kStage;
          const uint64_t da = kAMn ? umma_desc_mn128(sa) : umma_desc_k128(sa);
          const uint64_t db = kBMn ? umma_desc_mn128(sa + kOpBytes) : umma_desc_k128(sa + kOpBytes);
#pragma unroll
          for (int k = 0; k < kBlockK / 16; k++)          // 16 K columns are 32 bytes of a row, 16 K rows are 2 KB
            umma_bf16_pair(d, da + (uint64_t)(kAMn ? 128 * k : 2 * k), db + (uint64_t)(kBMn ? 128 * k : 2 * k), kIdesc, (j | k) != 0 ? 1u : 0u);
          umma_commit_pair(empty + s);
        }
        if (OP == kAdapt && sg.kind != kProduce) {
          factors_ready();
          int tm, tn;
          tile_at(sg.tile, m_tiles, n_tiles, tm, tn);
          const int* list = p.lists + (size_t)tm * kListStride;
          const int count = list[0], chunks = (p.R + kChunk - 1) / kChunk;
          for (int j = 0; j < count; j++) {
            for (int c = 0; c < chunks; c++, it++) {
              const int s = it % kStages;
              if (!gemm_wait(full + s, (it / kStages) & 1u, gw, 3)) goto done;
              mbar_test_cluster(full + s, (it / kStages) & 1u);      // through by now: takes what the other CTA's warps wrote
              tc_fence_after();
              const uint64_t da = umma_desc_k128(ring + s * kStage), db = umma_desc_k128(ring + s * kStage + kOpBytes);
              const int steps = (min(kChunk, p.R - c * kChunk) + 15) / 16;
              for (int k = 0; k < steps; k++) {
                umma_bf16_pair(d, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), kIdesc, 1u);
                umma_bf16_pair(d, da + (uint64_t)(4 + 2 * k), db + (uint64_t)(2 * k), kIdesc, 1u);
              }
              umma_commit_pair(empty + s);
            }
          }
        }
        umma_commit_pair(acc_full + a);
      }
    } else if (OP == kAdapt && lane == 0) {
      // The second CTA's warp hands its blocks of low-rank factors over to the leader: an arrival that releases at cluster scope waits for
      // all that its thread has in flight, which in the warps that copy would be the next blocks (1.6 us a block instead of 1.2).
      uint32_t next = 0, seen = 0;
      while (walk.next(sg)) {
        next += (uint32_t)sg.count;
        if (sg.kind == kProduce) continue;
        factors_ready();
        int tm, tn;
        tile_at(sg.tile, m_tiles, n_tiles, tm, tn);
        const int blocks = p.lists[(size_t)tm * kListStride] * ((p.R + kChunk - 1) / kChunk);
        for (int i = 0; i < blocks; i++, next++) {
          const int s = next % kStages;
          if (!gemm_wait(filled + s, seen >> s & 1u, gw, 1)) goto done;
          seen ^= 1u << s;
          mbar_arrive_cluster(cluster_addr(full + s, 0u));
        }
      }
    }
  } else if (OP == kAdapt && warp >= 10) {
    // ------------------------------------------------------------ blocks of low-rank factors
    const int lt = threadIdx.x - 320, chunks = (p.R + kChunk - 1) / kChunk;
    uint32_t next = 0;                          // ring stages before this one
    uint32_t seen = 0;                          // bit s: parity of the next grant of stage s (a stage is granted again only after its block is used up)
    for (uint32_t tile_i = 0; walk.next(sg); tile_i++) {
      next += (uint32_t)sg.count;
      if (sg.kind == kProduce) continue;
      factors_ready();
      int tm, tn;
      tile_at(sg.tile, m_tiles, n_tiles, tm, tn);
      const int m0 = tm * 256 + (int)crank * 128, n0 = tn * 256 + (int)crank * 128;
      const int* list = p.lists + (size_t)tm * kListStride;
      const int count = list[0];
      // which adapters of the list are left to the epilogue, before any stage is granted
      for (int j = warp - 10; j < count; j += 2) {
        const bool good = low_rank_finite<32>(p, list[1 + j], tn * 256, lane);
        if (lane == 0) skipped[j] = !good;
      }
      // this thread's 16 pieces of 16 bytes of a block: piece lt & 7 of rows lt / 8, + 8, ...
      int ids[16];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int row = m0 + (lt >> 3) + 8 * i;
        ids[i] = row < p.M ? p.ids[row] : -1;
      }
      low_rank_barrier();
      // Blocks are copied into their stages while up to three before them land and are handed over.  (With one before them and the
      // checks by both warps together a block took 1.9 us: 272 us for 128 rows of 128 adapters.)
      const int blocks = count * chunks;
      for (int k = 0; k < blocks + kLowAhead; k++) {
        if (k < blocks) {
          const int adapter = list[1 + k / chunks], c = k % chunks, s = (next + k) % kStages;
          if (!low_rank_all(gemm_wait(granted + s, seen >> s & 1u, gw, 1))) goto done;      // all of them or none
          seen ^= 1u << s;
          const bool good = !skipped[k / chunks];
          uint8_t *sa = ring + s * kStage, *sb = sa + kOpBytes;
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int r = (lt >> 3) + 8 * i;
            const bool copy = good && ids[i] == adapter;
            copy_or_zero(sa + r * 128 + (((lt & 7) ^ (r & 7)) << 4), copy ? p.v + ((size_t)(m0 + r) * chunks + c) * 64 + (lt & 7) * 8 : p.v, copy);
          }
          if (good) {
            if (lt == 0) tma_load_2d_pair(sb, &maps.low, c * kChunk, adapter * p.N + n0, cluster_addr(full + s, 0u));
          } else {
            if (lt == 0) unsafe_tile[tile_i % kVerdicts] = tile_i + 1u;      // before the arrival that the MMAs wait for
            for (int i = lt; i < kOpBytes / 16; i += kLowThreads) sts16(sb + 16 * i, make_uint4(0, 0, 0, 0));
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (k >= kLowAhead) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kLowAhead) : "memory");
          fence_smem_to_async();
          low_rank_barrier();
          if (lt == 0) {
            const int s = (next + k - kLowAhead) % kStages;
            if (leads) mbar_arrive_expect(full + s, skipped[(k - kLowAhead) / chunks] ? 0 : 2 * kOpBytes);
            else mbar_arrive(filled + s);
          }
        }
      }
      next += (uint32_t)blocks;
      low_rank_barrier();                       // `skipped` is read until here
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, side = (warp - 2) >> 2;
    uint8_t* slab = slabs + (warp - 2) * kSlab;
    uint32_t tile_i = 0;
    // chunk `j` (16 bytes) of this lane's row of the slab
    auto put = [&](int j, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
      sts16(slab + lane * 128 + ((j ^ (lane & 7)) << 4), make_uint4(w0, w1, w2, w3));
    };
    auto slab_free = [&]() {                   // its last store has been read
      if (lane == 0) bulk_wait_source_free<0>();
      __syncwarp();
    };
    auto slab_full = [&]() {
      fence_smem_to_async();
      __syncwarp();
    };
    // Two groups of 64 accumulator columns per tile: chunks of 32 columns group_chunk(g, 0) and (g, 1).  kGated: 32 gate columns and
    // the up columns that go with them.
    auto group_chunk = [&](int g, int which) { return OP == kGated ? 4 * which + 2 * side + g : 4 * side + 2 * g + which; };
    auto slot = [&](int cta, int c, int i) {   // float4 `i` of 32-column chunk `c`: a warp's rows are 512 contiguous bytes
      return reinterpret_cast<float4*>(p.partial) + (((size_t)cta * 8 + c) * 8 + i) * 128 + q * 32 + lane;
    };
    for (; walk.next(sg); tile_i++) {
      int tm, tn;
      tile_at(sg.tile, m_tiles, n_tiles, tm, tn);
      const uint32_t a = tile_i & 1u;
      const int row0 = tm * 256 + (int)crank * 128 + q * 32, n0 = tn * kTileN;
      const int first_col = n0 + (OP == kGated ? 64 : 128) * side;
      const bool mine = row0 + lane < p.M;
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + a * 256;
      uint32_t* const flag = p.flags + (size_t)blockIdx.x * kSplitFlags + (warp - 2);      // of this unit's slot
      float v[2][32], w[2][32];
      // what the units behind this one have left for a group
      auto load_shares = [&](int g) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int c = group_chunk(g, h);
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float4 f = __ldcg(slot(blockIdx.x + 2, c, i));
            w[h][4 * i] = f.x; w[h][4 * i + 1] = f.y; w[h][4 * i + 2] = f.z; w[h][4 * i + 3] = f.w;
          }
          for (int j = 2; j <= sg.others; j++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const float4 f = __ldcg(slot(blockIdx.x + 2 * j, c, i));
              w[h][4 * i] += f.x; w[h][4 * i + 1] += f.y; w[h][4 * i + 2] += f.z; w[h][4 * i + 3] += f.w;
            }
          }
        }
      };
      bool good = true;
      if (sg.kind == kProduce && lane == 0) good = gemm_flag_wait(flag, 0u, gw, 5);
      if (sg.kind == kFinish)
        for (int j = 1 + lane; j <= sg.others; j += 32) good = good && gemm_flag_wait(flag + 2 * kSplitFlags * j, 1u, gw, 6);
      if (!__all_sync(0xffffffffu, good)) break;
      __syncwarp();                                        // what one lane has acquired is ordered for the others too (a vote orders no memory)
      if (sg.kind == kFinish && mine) load_shares(0);      // in flight while the last K blocks run
      if (!__all_sync(0xffffffffu, gemm_wait(acc_full + a, (tile_i >> 1) & 1u, gw, 4))) break;
      tc_fence_after();
      if (row0 < p.M && first_col < p.N) {
        int slow = -1;                                     // kAdapt: this row's adapter is added here
        const __nv_bfloat16* vrow = nullptr;
        if (OP == kAdapt && sg.kind != kProduce) {
          const int id = mine ? p.ids[row0 + lane] : -1;
          if (unsafe_tile[tile_i % kVerdicts] == tile_i + 1u && id >= 0 && id < p.adapters && low_rank_unsafe(p, id, n0)) {
            factors_ready();
            slow = id;
            vrow = p.v + (size_t)(row0 + lane) * ((p.R + kChunk - 1) / kChunk * 64);
          }
        }
        uint32_t keep[16];                                 // kGated: h of the first group
#pragma unroll
        for (int g = 0; g < 2; g++) {
          const int col = first_col + (OP == kGated ? 32 : 64) * g;
          if (OP != kGated && col >= p.N) continue;
          tmem_ld32_issue(tbase + group_chunk(g, 0) * 32, v[0]);
          tmem_ld32_issue(tbase + group_chunk(g, 1) * 32, v[1]);
          tmem_ld_wait();
          if (sg.kind == kProduce) {
            if (mine) {
#pragma unroll
              for (int i = 0; i < 16; i++) {
                const float* f = v[i >> 3] + 4 * (i & 7);
                *slot(blockIdx.x, group_chunk(g, i >> 3), i & 7) = make_float4(f[0], f[1], f[2], f[3]);
              }
            }
            continue;
          }
          if (sg.kind == kFinish && mine) {
#pragma unroll
            for (int i = 0; i < 64; i++) v[i >> 5][i & 31] += w[i >> 5][i & 31];
          }
          if constexpr (OP == kGated) {
            if (p.want_pre && col < p.N) {
#pragma unroll
              for (int which = 0; which < 2; which++) {
                slab_free();
#pragma unroll
                for (int j = 0; j < 8; j++) {
                  const float* f = v[which] + 4 * j;
                  put(j, __float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
                }
                slab_full();
                if (lane == 0) { tma_store_3d(&maps.pre, col, which, row0, slab); bulk_commit(); }
              }
            }
            if (p.act == FP4AR_ACT_SILU) {
#pragma unroll
              for (int i = 0; i < 32; i++) v[0][i] = act_value<FP4AR_ACT_SILU>(v[0][i]) * v[1][i];
            } else if (p.act == FP4AR_ACT_GELU) {
#pragma unroll
              for (int i = 0; i < 32; i++) v[0][i] = act_value<FP4AR_ACT_GELU>(v[0][i]) * v[1][i];
            } else {
#pragma unroll
              for (int i = 0; i < 32; i++) v[0][i] = act_value<FP4AR_ACT_GELU_TANH>(v[0][i]) * v[1][i];
            }
            if (g == 0) {
#pragma unroll
              for (int i = 0; i < 16; i++) keep[i] = pack_bf16(v[0][2 * i], v[0][2 * i + 1]);
              if (sg.kind == kFinish && mine) load_shares(1);
              continue;
            }
            slab_free();
#pragma unroll
            for (int j = 0; j < 4; j++) {
              put(j, keep[4 * j], keep[4 * j + 1], keep[4 * j + 2], keep[4 * j + 3]);
              const float* f = v[0] + 8 * j;
              put(4 + j, pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
            }
            slab_full();
            if (lane == 0) { tma_store_2d(&maps.out, first_col, row0, slab); bulk_commit(); }
          } else {
            if constexpr (OP == kAdapt) {
              if (slow >= 0) {
#pragma unroll
                for (int i = 0; i < 64; i++)
                  if (col + i < p.N) v[i >> 5][i & 31] += low_rank_dot(vrow, p.b + ((size_t)slow * p.N + col + i) * p.R, p.R);
              }
              __syncwarp();
            }
            slab_free();
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const float* f = v[j >> 2] + 8 * (j & 3);
              put(j, pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
            }
            slab_full();
            if (lane == 0) { tma_store_2d(&maps.out, col, row0, slab); bulk_commit(); }
            if (g == 0 && sg.kind == kFinish && mine) load_shares(1);
          }
        }
      }
      tc_fence_before();
      __syncwarp();                                        // every lane has its accumulators and shares in registers
      if (lane == 0) mbar_arrive_cluster_relaxed(cluster_addr(acc_empty + a, 0u));
      if (sg.kind == kProduce && lane == 0) { __threadfence(); st_release_gpu(flag, 1u); }
      if (sg.kind == kFinish)
        for (int j = 1 + lane; j <= sg.others; j += 32) st_release_gpu(flag + 2 * kSplitFlags * j, 0u);
    }
    if (lane == 0) bulk_wait_done<0>();
  }
done:
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0u) {
    // what was issued lands before the CTA leaves: its own copies under the leader's barriers, the MMAs under `settled`
    if (leads && threadIdx.x == 0)
      for (uint32_t i = issued > (uint32_t)kStages ? issued - kStages : 0u; i < issued; i++) gemm_settle(full + i % kStages, (i / kStages) & 1u);
    if (!leads && threadIdx.x == 0)
      for (int w = 0; w < 2000; w++) __nanosleep(1000);
    if (leads && threadIdx.x == 32) {
      umma_commit_pair(settled);
      gemm_settle(settled, 0u);
    }
    __syncthreads();
  }
  cluster_sync_all();     // neither CTA frees TMEM or leaves while the other's MMAs, commits or arrivals may still touch it
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---- host side ----
// A BF16 matrix of `rows` rows, `cols` contiguous columns; box of 64 columns x box_rows.
inline bool map_2d(CUtensorMap* m, const void* base, long rows, long cols, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, one[2] = {1, 1};
  return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}
// [rows][2][cols] FP32: the two projections of every row, each clipped at its own width
inline bool map_pre(CUtensorMap* m, const void* base, long rows, long cols) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, 2, (cuuint64_t)rows}, strides[2] = {(cuuint64_t)cols * 4, (cuuint64_t)cols * 8};
  const cuuint32_t box[3] = {32, 1, 32}, one[3] = {1, 1, 1};
  return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

constexpr unsigned long long kWaitLimitNs = 2000000000ull;

// How many units share the tiles that are cut (0: none).  A block takes a unit 0.3 us; writing, reading and adding the partials costs
// about 10 us, so tiles are cut where that saves the units 48 blocks each on average.  (h of 1031 x 1368, K = 6144: 25 idle blocks of 96,
// 37.5 us whole, 40.9 cut; 2048 x 2048, K = 8192: 35 of 256, 98.4 and 104.9; 4096 x 2048, K = 6144: 52 of 384, 148.5 and 146.7, K = 8192: 69
// of 512, 198.1 and 190.5; 256 x 2048, K = 4096: 50 of 64, 29.7 and 29.2, K = 8192: 100 of 128, 49.7 and 33.3.)
inline int cut_units(int tiles, int kblocks, int units) {
  const long long waves = (tiles + units - 1) / units, idle = (waves * units - tiles) * kblocks / units;
  if (idle < 48) return 0;
  if (tiles >= units) return units;
  const long long ranges = (long long)tiles * kblocks / 8;
  return ranges <= tiles ? 0 : ranges < units ? (int)ranges : units;
}

template <int OP>
int launch_pair_gemm(const Maps& maps, Params p, cudaStream_t stream) {
  static std::atomic<int> resident[64];          // pairs that can be resident together, 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cuda_fail();
  p.status = gemm_status_word();
  if (!p.status) return cuda_fail();
  p.timeout_ns = kWaitLimitNs;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.blockDim = dim3(kThreads<OP>);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int fits = resident[dev].load(std::memory_order_acquire);
  if (!fits) {
    if (cudaFuncSetAttribute(pair_gemm_kernel<OP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) != cudaSuccess) return cuda_fail();
    cfg.gridDim = dim3(device_sm_count() & ~1);
    if (cudaOccupancyMaxActiveClusters(&fits, pair_gemm_kernel<OP>, &cfg) != cudaSuccess || fits < 1) return cuda_fail();
    resident[dev].store(fits, std::memory_order_release);
  }
  constexpr int kTileN = OP == kGated ? 128 : 256;
  const long tiles = ((long)p.M + 255) / 256 * (((long)p.N + kTileN - 1) / kTileN);
  if (tiles > 0x7fff0000L) return FP4AR_ERR_ARGUMENT;
  const int whole = tiles < fits ? (int)tiles : fits;
  p.cut_units = cut_units((int)tiles, p.kblocks, fits);
  int units = p.cut_units > whole ? p.cut_units : whole;
  std::optional<SplitSpace> space;
  if (p.cut_units) {
    try {
      space.emplace(stream);
      p.partial = space->partial();
      p.flags = space->flags();
    } catch (...) {}                       // no host memory for it: whole tiles
    if (!p.partial) { p.cut_units = 0; units = whole; }
  }
  cfg.gridDim = dim3(2 * units);
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, pair_gemm_kernel<OP>, maps, p) != cudaSuccess) return cuda_fail();
  return cuda_check_launch();
}

inline bool aligned16(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) == 0;
}
// Tensor map extents and coordinates are 32-bit
inline bool extents_ok(long long a, long long b) { return a <= 0x7fffff00LL && b <= 0x7fffff00LL; }

}  // namespace layer
}  // namespace fp4ar
