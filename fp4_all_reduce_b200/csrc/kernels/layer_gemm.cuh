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
//   warps 2-5   epilogue: tcgen05.ld, activation, BF16, a 32 x 64 slab per warp in swizzled shared memory, TMA store
// Ragged sizes need no code in the main loop: tensor maps fill with zeros beyond their extents and stores are clipped.
//
// MN-major tiles: a box of 64 (outer index, 128 bytes, swizzled) x 64 K rows is 8 KB; a tile of 128 is two boxes.  In the
// descriptor the leading offset is the distance between boxes (8192), the stride offset that between groups of 8 K rows (1024).
#pragma once
#include <atomic>
#include <cstring>
#include <cuda_bf16.h>
#include "../include/fp4ar_layer.h"
#include "../include/fp4ar_tensor.cuh"
#include "activation.cuh"
#include "host_util.h"
#include "tensor_map.h"

namespace fp4ar {
namespace layer {

enum : int { kGated = 0, kInput = 1, kWeight = 2, kAdapt = 3 };

constexpr int kRowsCta = 128, kBlockK = 64, kHalf = 128, kStages = 6, kThreads = 192;
constexpr int kOpBytes = kRowsCta * kBlockK * 2;               // 16 KB of A, 16 KB of B per CTA and stage
constexpr int kStage = 2 * kOpBytes;
constexpr int kSlab = 32 * 64 * 2;                             // 32 rows x 64 BF16 columns, one warp's store
constexpr int kSlabs = 4 * 2 * kSlab;                          // two per epilogue warp
constexpr int kSmemBytes = kStages * kStage + kSlabs + 256 + 1024;
constexpr int kListStride = 260;                               // per 256-row tile: count, then up to 256 adapters (16-byte pitch)
constexpr int kChunk = 32;                                     // ranks per block of low-rank factors

struct Params {
  int M, N;                 // rows and columns of the output (kGated: columns of h)
  int kblocks;
  int act;
  bool want_pre;
  // adapters
  int R, adapters;
  const int* ids;           // [M]
  const float* v;           // [M][R] scaled x A^T, FP32
  const int* lists;         // [row tiles][kListStride]
  const unsigned char* unsafe;   // [adapters] 1: B holds infinities or NaN
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

// ---- Adapters.  y_i = x_i W^T + sum_r V[i][r] B_a[:, r], a = ids[i].  A 256-row tile has a list of the adapters its rows use; for
// each of them and every 32 ranks follows one more block of the same accumulation: A is V of the rows that have this adapter and
// zero elsewhere, as two BF16 halves (columns 0-31 the rounded value, 32-63 what the rounding left, so V counts with 16 bits), B is
// B_a [128 columns x ranks] twice.  The producer warp writes the A block itself; W's blocks keep coming by TMA.
// 0 x infinity would leak one request's broken adapter into the rows of others, so adapters whose B is not finite are
// marked beforehand and left out here; the epilogue adds them to their own rows by plain dot products.
__device__ __forceinline__ void write_low_rank_block(uint8_t* dst, const Params& p, int adapter, int chunk, int row0, int lane) {
  const int ranks = min(kChunk, p.R - chunk * kChunk);         // a multiple of 8
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = i * 32 + lane, row = row0 + r;
    const bool mine = row < p.M && p.ids[row] == adapter;
    const float* v = p.v + (size_t)row * p.R + chunk * kChunk;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
      if (mine && 8 * j < ranks) {
        const float4 f0 = *reinterpret_cast<const float4*>(v + 8 * j), f1 = *reinterpret_cast<const float4*>(v + 8 * j + 4);
        const float f[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          hi[e] = pack_bf16(f[2 * e], f[2 * e + 1]);
          const float h0 = bf16_lo(hi[e]), h1 = bf16_hi(hi[e]);
          // what is not finite stays in the first half alone
          lo[e] = pack_bf16(fabsf(h0) <= 3.4e38f ? f[2 * e] - h0 : 0.0f, fabsf(h1) <= 3.4e38f ? f[2 * e + 1] - h1 : 0.0f);
        }
      }
      uint8_t* line = dst + r * 128;
      sts16(line + ((j ^ (r & 7)) << 4), make_uint4(hi[0], hi[1], hi[2], hi[3]));
      sts16(line + (((4 + j) ^ (r & 7)) << 4), make_uint4(lo[0], lo[1], lo[2], lo[3]));
    }
  }
}

static __device__ __noinline__ float low_rank_dot(const float* v, const __nv_bfloat16* b, int R) {
  float s = 0.0f;
  for (int r = 0; r < R; r++) s = fmaf(v[r], __bfloat162float(b[r]), s);
  return s;
}

template <int OP>
__global__ void __launch_bounds__(kThreads, 1)
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
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(settled + 1);
  volatile uint32_t* abort_flag = tmem_holder + 1;
  uint32_t issued = 0;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m_tiles = (p.M + 255) / 256, n_tiles = (p.N + kTileN - 1) / kTileN, tiles = m_tiles * n_tiles;
  const uint32_t crank = cluster_cta_rank();
  const bool leads = crank == 0u;
  const int unit = blockIdx.x / 2, units = gridDim.x / 2;

  if (threadIdx.x == 0) {
    // kAdapt: both producers announce a stage, since both may write into it themselves
    for (int s = 0; s < kStages; s++) { mbar_init(full + s, OP == kAdapt ? 2 : 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; a++) { mbar_init(acc_full + a, 1); mbar_init(acc_empty + a, 256); }
    mbar_init(settled, 1);
    *abort_flag = 0u;
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

  pdl_wait_prior_grids();
  pdl_release_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------ producer (kAdapt: the whole warp)
    if (OP == kAdapt || lane == 0) {
      auto stage_free = [&](int s) {
        const bool ok = gemm_wait(empty + s, ((issued / kStages) & 1u) ^ 1u, gw, 1);
        return OP == kAdapt ? (bool)__all_sync(0xffffffffu, ok) : ok;
      };
      for (int t = unit; t < tiles; t += units) {
        int tm, tn;
        tile_at(t, m_tiles, n_tiles, tm, tn);
        const int m0 = tm * 256 + (int)crank * 128;
        const int n0 = OP == kGated ? tn * 128 + (int)crank * p.N : tn * 256 + (int)crank * 128;
        for (int kb = 0; kb < p.kblocks; kb++, issued++) {
          const int s = issued % kStages;
          if (!stage_free(s)) goto done;
          if (lane == 0) {
            uint8_t *sa = ring + s * kStage, *sb = sa + kOpBytes;
            const uint32_t lead_full = cluster_addr(full + s, 0u);
            if (leads) mbar_arrive_expect(full + s, 2 * kStage);
            else if (OP == kAdapt) mbar_arrive_cluster(lead_full);
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
        }
        if constexpr (OP == kAdapt) {
          const int* list = p.lists + (size_t)tm * kListStride;
          const int count = list[0], chunks = (p.R + kChunk - 1) / kChunk;
          for (int j = 0; j < count; j++) {
            const int adapter = list[1 + j];
            if (p.unsafe[adapter]) continue;
            for (int c = 0; c < chunks; c++, issued++) {
              const int s = issued % kStages;
              if (!stage_free(s)) goto done;
              uint8_t *sa = ring + s * kStage, *sb = sa + kOpBytes;
              write_low_rank_block(sa, p, adapter, c, m0, lane);
              fence_smem_to_async();
              __syncwarp();
              if (lane == 0) {
                const uint32_t lead_full = cluster_addr(full + s, 0u);
                if (leads) mbar_arrive_expect(full + s, 2 * kOpBytes);
                else mbar_arrive_cluster(lead_full);
                tma_load_2d_pair(sb, &maps.low, c * kChunk, adapter * p.N + n0, lead_full);
              }
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && leads) {
      uint32_t it = 0, tile_i = 0;
      auto stage_ready = [&](int s, uint32_t round) {
        if constexpr (OP != kAdapt) return gemm_wait(full + s, round & 1u, gw, 3);
        // the second wait takes what the other CTA's producer wrote, at cluster scope
        else return gemm_wait(full + s, round & 1u, gw, 3) && mbar_test_cluster(full + s, round & 1u);
      };
      for (int t = unit; t < tiles; t += units, tile_i++) {
        const uint32_t a = tile_i & 1u;
        if (!gemm_wait(acc_empty + a, ((tile_i >> 1) & 1u) ^ 1u, gw, 2)) goto done;
        tc_fence_after();
        const uint32_t d = tmem_base + a * 256;
        for (int kb = 0; kb < p.kblocks; kb++, it++) {
          const int s = it % kStages;
          if (!stage_ready(s, it / kStages)) goto done;
          tc_fence_after();
          const uint8_t* sa = ring + s * kStage;
          const uint64_t da = kAMn ? umma_desc_mn128(sa) : umma_desc_k128(sa);
          const uint64_t db = kBMn ? umma_desc_mn128(sa + kOpBytes) : umma_desc_k128(sa + kOpBytes);
#pragma unroll
          for (int k = 0; k < kBlockK / 16; k++)          // 16 K columns are 32 bytes of a row, 16 K rows are 2 KB
            umma_bf16_pair(d, da + (uint64_t)(kAMn ? 128 * k : 2 * k), db + (uint64_t)(kBMn ? 128 * k : 2 * k), kIdesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit_pair(empty + s);
        }
        if constexpr (OP == kAdapt) {
          int tm, tn;
          tile_at(t, m_tiles, n_tiles, tm, tn);
          const int* list = p.lists + (size_t)tm * kListStride;
          const int count = list[0], chunks = (p.R + kChunk - 1) / kChunk;
          for (int j = 0; j < count; j++) {
            if (p.unsafe[list[1 + j]]) continue;
            for (int c = 0; c < chunks; c++, it++) {
              const int s = it % kStages;
              if (!stage_ready(s, it / kStages)) goto done;
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
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;
    uint8_t* my_slabs = slabs + q * 2 * kSlab;
    uint32_t tile_i = 0, stores = 0;
    // This lane's 32 values, columns 32 `half` .. + 31 of its row of a slab.
    auto put = [&](uint8_t* slab, int half, const float* v) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        sts16(slab + lane * 128 + (((half * 4 + j) ^ (lane & 7)) << 4),
              make_uint4(pack_bf16(v[8 * j], v[8 * j + 1]), pack_bf16(v[8 * j + 2], v[8 * j + 3]), pack_bf16(v[8 * j + 4], v[8 * j + 5]),
                         pack_bf16(v[8 * j + 6], v[8 * j + 7])));
    };
    auto next_slab = [&]() {                   // of the two, the one whose store has been read
      if (lane == 0) bulk_wait_source_free<1>();
      __syncwarp();
      return my_slabs + (stores++ & 1u) * kSlab;
    };
    for (int t = unit; t < tiles; t += units, tile_i++) {
      int tm, tn;
      tile_at(t, m_tiles, n_tiles, tm, tn);
      const uint32_t a = tile_i & 1u;
      const int row0 = tm * 256 + (int)crank * 128 + q * 32, n0 = tn * kTileN;
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + a * 256;
      if (!__all_sync(0xffffffffu, gemm_wait(acc_full + a, (tile_i >> 1) & 1u, gw, 4))) break;
      tc_fence_after();
      if (row0 < p.M) {
        float v[2][32];
        if (OP != kGated || p.want_pre) {
          // all 256 accumulator columns as they are
          int slow = -1;
          const float* vrow = nullptr;
          if constexpr (OP == kAdapt) {
            const int row = row0 + lane;
            const int id = row < p.M ? p.ids[row] : -1;
            if (id >= 0 && id < p.adapters && p.unsafe[id]) { slow = id; vrow = p.v + (size_t)row * p.R; }
          }
          for (int c = 0; c < 4; c++) {
            const int col = OP == kGated ? n0 + (c & 1) * 64 : n0 + c * 64;
            if (col >= p.N) continue;
            tmem_ld32_issue(tbase + c * 64, v[0]);
            tmem_ld32_issue(tbase + c * 64 + 32, v[1]);
            uint8_t* slab = next_slab();
            tmem_ld_wait();
            if constexpr (OP == kAdapt) {
              if (slow >= 0) {
#pragma unroll
                for (int i = 0; i < 64; i++)
                  if (col + i < p.N) v[i >> 5][i & 31] += low_rank_dot(vrow, p.b + ((size_t)slow * p.N + col + i) * p.R, p.R);
              }
            }
            put(slab, 0, v[0]);
            put(slab, 1, v[1]);
            fence_smem_to_async();
            __syncwarp();
            if (lane == 0) {
              if constexpr (OP == kGated) tma_store_3d(&maps.pre, col, c >> 1, row0, slab);
              else tma_store_2d(&maps.out, col, row0, slab);
              bulk_commit();
            }
          }
        }
        if constexpr (OP == kGated) {
          for (int c = 0; c < 2; c++) {
            const int col = n0 + c * 64;
            if (col >= p.N) continue;
            uint8_t* slab = next_slab();
            for (int half = 0; half < 2; half++) {
              tmem_ld32_issue(tbase + c * 64 + half * 32, v[0]);
              tmem_ld32_issue(tbase + 128 + c * 64 + half * 32, v[1]);
              tmem_ld_wait();
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
              put(slab, half, v[0]);
            }
            fence_smem_to_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&maps.out, col, row0, slab);
              bulk_commit();
            }
          }
        }
      }
      tc_fence_before();
      mbar_arrive_cluster(cluster_addr(acc_empty + a, 0u));
      __syncwarp();
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
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, one[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// [rows][2][cols]: the two projections of every row, each clipped at its own width
inline bool map_pre(CUtensorMap* m, const void* base, long rows, long cols) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, 2, (cuuint64_t)rows}, strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)cols * 4};
  const cuuint32_t box[3] = {64, 1, 32}, one[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr unsigned long long kWaitLimitNs = 2000000000ull;

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
  cfg.blockDim = dim3(kThreads);
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
  if (tiles > 0x7fffffffL) return FP4AR_ERR_ARGUMENT;
  const int units = tiles < fits ? (int)tiles : fits;
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
