// The same products for few rows, where the time is that of reading the weights once.
//
// The operands change sides: 128 rows of W (kInput: columns) are the M of the tcgen05 product and the rows of x its N (16 .. 256), so
// next to nothing is multiplied for rows that are not there.  A CTA of its own for every 128 rows of W would leave SMs idle and the
// others with a long chain of K blocks, so a cluster of up to eight CTAs cuts K: each leaves its FP32 sums in shared memory, and all
// of them add up a share of the outputs, in the order of the CTAs.  Up to 128 rows two CTAs fit an SM, and one's set-up and sums run
// under the other's loads (WIDE = false); more rows take groups of up to 256, a CTA for each (WIDE).
// Bound by the reads of W, by launch and latency where W is small: F = 8192, K = 6144 (201 MB), 16 rows 35 us, 5.8 TB/s; F = 2048 (50 MB), 1 row
// 11.6 us, 48 rows 13.3 (one CTA per tile, whole K loops: 39 and 40; tiles of 256 rows of x: 28 and 27); N = 6144, K = 2048, rank 16
// (26 and 38 MB): 1 row 8.6, 64 rows of 48 adapters 14.5.
//   kGated   the 128 rows are 64 gate rows and the 64 up rows that go with them: their product is taken where the sums meet
//   kAdapt   the low-rank parts of the outputs that a CTA adds up are computed by the epilogue warps while the weights stream in, by
//            plain FP32 products with V.  V comes from a launch before this one; only those warps wait for it (see below)
#pragma once
#include "layer_gemm.cuh"

namespace fp4ar {
namespace layer {

constexpr int kNarrowRows = 128, kFewStagesMax = 8;
template <int OP> constexpr int kFewThreads = OP == kAdapt ? 320 : 192;      // kAdapt: four more warps for the low-rank parts

struct FewParams {
  int M, N, kblocks, split, stages, tokens, groups;      // tokens: rows of a group, a multiple of 16; N: columns of the output
  int act;
  __nv_bfloat16* out;
  float* pre;                                    // kGated, optional [M][2 N]
  // kAdapt, as in Params
  int R, adapters, low_offset;
  const int* ids;
  const __nv_bfloat16* v;
  const __nv_bfloat16* b;
  StatusWords* status;
  unsigned long long timeout_ns;
};

__device__ __forceinline__ float4 cluster_ld4(uint32_t addr) {
  float4 f;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(addr));
  return f;
}
__device__ __forceinline__ void prefetch_tile(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ float act_any(int act, float g) {
  return act == FP4AR_ACT_SILU ? act_value<FP4AR_ACT_SILU>(g) : act == FP4AR_ACT_GELU ? act_value<FP4AR_ACT_GELU>(g) : act_value<FP4AR_ACT_GELU_TANH>(g);
}

template <int OP, bool WIDE>
__global__ void __launch_bounds__(kFewThreads<OP>, WIDE ? 1 : 2)
few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ FewParams p) {
  static_assert(OP == kGated || OP == kInput || (OP == kAdapt && !WIDE), "products with W");
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kFewStagesMax], empty[kFewStagesMax], acc_full;
  __shared__ uint32_t tmem_holder;
  __shared__ volatile uint32_t abort_flag;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* part = reinterpret_cast<float*>(ring);  // [tokens][128], once the ring has been read
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the groups of one tile are neighbours: its weights cross HBM once
  const int crank = blockIdx.x % p.split, group = blockIdx.x / p.split % p.groups, tile = blockIdx.x / p.split / p.groups;
  const int first = group * p.tokens, rows = min(p.tokens, p.M - first);
  const int stage_bytes = kOpBytes + p.tokens * 128;
  constexpr uint32_t cols = WIDE ? 256 : 128;
  if (tid == 0) {
    for (int s = 0; s < p.stages; s++) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    mbar_init(&acc_full, 1);
    abort_flag = 0u;
    mbar_init_fence();
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
  }
  if (warp == 1) { tmem_alloc(&tmem_holder, cols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_holder;
  GemmWait gw{&abort_flag, p.status, p.timeout_ns};
  // kAdapt: the launch before this one lets it start only after its own wait, so everything before that one is complete here; what
  // that one itself writes (V) is waited for where it is read.
  // The first weights are asked into L2 before that wait: whoever writes them before it writes them there.
  const int kb0 = p.kblocks * crank / p.split, kb1 = p.kblocks * (crank + 1) / p.split;
  const int row0 = OP == kGated ? tile * 64 : tile * 128, row1 = OP == kGated ? p.N + row0 : row0 + 64;
  if (warp == 0 && lane < p.stages && kb0 + lane < kb1) {
    const int k = (kb0 + lane) * kBlockK;
    prefetch_tile(&map_w, OP == kInput ? row0 : k, OP == kInput ? k : row0);
    prefetch_tile(&map_w, OP == kInput ? row1 : k, OP == kInput ? k : row1);
  }
  if (OP != kAdapt) pdl_wait_prior_grids();
  pdl_release_dependents();

  // this CTA's share of the outputs, in groups of four
  const int items = rows * (OP == kGated ? 16 : 32), item0 = items * crank / p.split, item1 = items * (crank + 1) / p.split;
  float4* lows = reinterpret_cast<float4*>(ring + p.low_offset);
  int issued = 0;
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; kb++, issued++) {
        const int s = issued % p.stages;
        if (!gemm_wait(empty + s, ((issued / p.stages) & 1u) ^ 1u, gw, 1)) break;
        uint8_t* at = ring + s * stage_bytes;
        mbar_arrive_expect(full + s, stage_bytes);
        if constexpr (OP == kInput) {
          tma_load_2d(at, &map_w, row0, kb * kBlockK, full + s);
          tma_load_2d(at + kOpBytes / 2, &map_w, row1, kb * kBlockK, full + s);
        } else {
          tma_load_2d(at, &map_w, kb * kBlockK, row0, full + s);
          tma_load_2d(at + kOpBytes / 2, &map_w, kb * kBlockK, row1, full + s);
        }
        tma_load_2d(at + kOpBytes, &map_x, kb * kBlockK, first, full + s);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((OP == kInput ? 1u : 0u) << 15) | ((uint32_t)(p.tokens >> 3) << 17) | ((128u >> 4) << 24);
      for (int it = 0; it < kb1 - kb0; it++) {
        const int s = it % p.stages;
        if (!gemm_wait(full + s, (it / p.stages) & 1u, gw, 3)) break;
        tc_fence_after();
        const uint8_t* sw = ring + s * stage_bytes;
        const uint64_t da = OP == kInput ? umma_desc_mn128(sw) : umma_desc_k128(sw), db = umma_desc_k128(ring + s * stage_bytes + kOpBytes);
#pragma unroll
        for (int k = 0; k < kBlockK / 16; k++) umma_bf16(tmem_base, da + (uint64_t)((OP == kInput ? 128 : 2) * k), db + (uint64_t)(2 * k), idesc, (it | k) != 0 ? 1u : 0u);
        umma_commit(empty + s);
      }
      umma_commit(&acc_full);
    }
  } else {
    if constexpr (OP == kAdapt) {
      // The low-rank parts of this CTA's share of the outputs, a warp for each row of x.  B_a is read as it lies: `width` lanes have 16
      // bytes each of one of its rows (eight ranks, whose V stay in registers), so a warp's load is 512 contiguous bytes, and the
      // lanes of a row add up by shuffles.  (A lane with four rows of its own: 24 us instead of 5 at 64 rows of 16 adapters,
      // K = 8192, R = 64, where the product alone takes 25.)  The lines
      // are asked for before V is there.
      const int pieces = p.R / 8, width = pieces > 8 ? 16 : pieces > 4 ? 8 : pieces > 2 ? 4 : pieces, per_load = 32 / width;
      const int sub = lane % width, line = (p.R + kChunk - 1) / kChunk * 64;
      auto share_of = [&](int m, int& from, int& to) -> const uint4* {      // B_a from row `row0` on, rows [from, to) of the tile
        from = max(4 * item0 - m * 128, 0);
        to = min(min(4 * item1 - m * 128, 128), p.N - row0);
        const int id = p.ids[first + m];
        return id >= 0 && id < p.adapters ? reinterpret_cast<const uint4*>(p.b + ((size_t)id * p.N + row0) * p.R) : nullptr;
      };
      const int m0 = item0 / 32 + warp - 2, m1 = (item1 + 31) / 32;
      int from, to;
      for (int m = m0; m < m1; m += 8)
        if (const uint4* b = share_of(m, from, to))
          for (int o = from * pieces + lane * 8; o < to * pieces; o += 32 * 8) asm volatile("prefetch.global.L2 [%0];" ::"l"(b + o));
      pdl_wait_prior_grids();
      for (int m = m0; m < m1; m += 8) {
        const uint4* b = share_of(m, from, to);
        float* low = reinterpret_cast<float*>(lows) + m * 128 - 4 * item0;
        if (!b) {
          for (int r = from + lane; r < to; r += 32) low[r] = 0.0f;
          continue;
        }
        float v[8];
        const int piece = min(sub, pieces - 1);          // (lanes beyond the last piece read it too and add nothing)
        const uint4* at = reinterpret_cast<const uint4*>(p.v + (size_t)(first + m) * line + piece / 4 * 64 + piece % 4 * 8);
        const uint4 hi = __ldcg(at), lo = __ldcg(at + kChunk / 8);
        const uint32_t h4[4] = {hi.x, hi.y, hi.z, hi.w}, l4[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          v[2 * e] = bf16_lo(h4[e]) + bf16_lo(l4[e]);
          v[2 * e + 1] = bf16_hi(h4[e]) + bf16_hi(l4[e]);
        }
        for (int r0 = from; r0 < to; r0 += 8 * per_load) {                                   // eight loads in flight
          const int r = r0 + lane / width;
          uint4 w[8];
          float s[8];
#pragma unroll
          for (int k = 0; k < 8; k++) w[k] = __ldg(b + min(r + k * per_load, to - 1) * pieces + piece);
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const uint32_t w4[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
            s[k] = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) s[k] = fmaf(v[2 * e + 1], bf16_hi(w4[e]), fmaf(v[2 * e], bf16_lo(w4[e]), s[k]));
            if (sub >= pieces) s[k] = 0.0f;
          }
          for (int o = width / 2; o; o >>= 1) {
#pragma unroll
            for (int k = 0; k < 8; k++) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
          }
#pragma unroll
          for (int k = 0; k < 8; k++)
            if (sub == 0 && r + k * per_load < to) low[r + k * per_load] = s[k];
        }
      }
    }
    const int q = warp & 3;
    if (warp < 6 && __all_sync(0xffffffffu, gemm_wait(&acc_full, 0u, gw, 4)) && !__any_sync(0xffffffffu, abort_flag != 0u)) {
      tc_fence_after();
      for (int c = 0; c < p.tokens; c += 16) {
        float v[16];
        tmem_ld16_issue(tmem_base + ((uint32_t)(q * 32) << 16) + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; i++) part[(c + i) * 128 + q * 32 + lane] = v[i];
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (abort_flag != 0u) {
    if (tid == 0)
      for (int i = max(0, issued - p.stages); i < issued; i++) gemm_settle(full + i % p.stages, (i / p.stages) & 1);
    if (tid == 32) gemm_settle(&acc_full, 0u);       // committed behind every MMA issued
    __syncthreads();
  }
  if (p.split > 1) cluster_sync_all();
  // Four neighbouring outputs of a row at a time.
  const uint32_t base = smem_addr(part);
  auto sum4 = [&](int at) {
    if (p.split == 1) return *reinterpret_cast<const float4*>(part + at);
    float4 f[8];                                     // all of them in flight
#pragma unroll
    for (int d = 0; d < 8; d++)
      if (d < p.split) {
        uint32_t a;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(base + at * 4), "r"(d));
        f[d] = cluster_ld4(a);
      }
#pragma unroll
    for (int d = 1; d < 8; d++)
      if (d < p.split) { f[0].x += f[d].x; f[0].y += f[d].y; f[0].z += f[d].z; f[0].w += f[d].w; }
    return f[0];
  };
  if constexpr (OP == kGated) {
    for (int i = item0 + tid; i < item1; i += kFewThreads<OP>) {
      const int c = i % 16 * 4, f = row0 + c;
      if (f >= p.N) continue;
      const float4 g = sum4(i / 16 * 128 + c), u = sum4(i / 16 * 128 + 64 + c);
      const int m = first + i / 16;
      if (p.pre) {
        *reinterpret_cast<float4*>(p.pre + (size_t)m * 2 * p.N + f) = g;
        *reinterpret_cast<float4*>(p.pre + ((size_t)m * 2 + 1) * p.N + f) = u;
      }
      const uint2 h = make_uint2(pack_bf16(act_any(p.act, g.x) * u.x, act_any(p.act, g.y) * u.y),
                                 pack_bf16(act_any(p.act, g.z) * u.z, act_any(p.act, g.w) * u.w));
      *reinterpret_cast<uint2*>(p.out + (size_t)m * p.N + f) = h;
    }
  } else {
    for (int i = item0 + tid; i < item1; i += kFewThreads<OP>) {
      const int c = i % 32 * 4, n = row0 + c;
      if (n >= p.N) continue;
      const float4 s = sum4(i / 32 * 128 + c), low = OP == kAdapt ? lows[i - item0] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      *reinterpret_cast<uint2*>(p.out + (size_t)(first + i / 32) * p.N + n) = make_uint2(pack_bf16(s.x + low.x, s.y + low.y), pack_bf16(s.z + low.z, s.w + low.w));
    }
  }
  if (p.split > 1) cluster_sync_relaxed();           // a CTA's sums are read until here
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, cols);
  }
}

// Stands in for few_rows_kernel where the runtime is asked how many clusters fit: for a kernel that allocates TMEM it answers with one CTA
// an SM whatever the kernel takes (two were seen to run side by side).
template <int OP, bool WIDE>
__global__ void __launch_bounds__(kFewThreads<OP>, WIDE ? 1 : 2) few_rows_room_kernel() {}

// `w` has `rows` rows: 2 N of K columns (kGated), N (kAdapt), K rows of N columns (kInput).
template <int OP, bool WIDE>
int launch_few_rows(const void* w, long rows, const void* x, int K, FewParams p, cudaStream_t stream) {
  constexpr int kBudget = (WIDE ? 220 : 110) * 1024;  // of dynamic shared memory
  static std::atomic<int> raised[64];
  static std::atomic<int> clusters[64][9];           // how many clusters of a size can be resident
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cuda_fail();
  if (!raised[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(few_rows_kernel<OP, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBudget) != cudaSuccess ||
        cudaFuncSetAttribute(few_rows_kernel<OP, WIDE>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess ||
        cudaFuncSetAttribute(few_rows_room_kernel<OP, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBudget + 1024) != cudaSuccess)
      return cuda_fail();
    for (int c = 1; c <= 8; c++) {
      cudaLaunchConfig_t cfg;
      memset(&cfg, 0, sizeof(cfg));
      cfg.gridDim = dim3(64 * c);
      cfg.blockDim = dim3(kFewThreads<OP>);
      cfg.dynamicSmemBytes = kBudget + 256;          // and the barriers
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = c; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, few_rows_room_kernel<OP, WIDE>, &cfg) != cudaSuccess) return cuda_fail();
      clusters[dev][c].store(n, std::memory_order_release);
    }
    raised[dev].store(1, std::memory_order_release);
  }
  p.status = gemm_status_word();
  if (!p.status) return cuda_fail();
  p.timeout_ns = kWaitLimitNs;
  p.kblocks = (K + 63) / 64;
  const int most = WIDE ? 256 : kNarrowRows, per_tile = OP == kGated ? 64 : 128;
  long tiles;
  int lows, sums;                                    // bytes for the low-rank parts and for the sums (which take the ring's place)
  for (int g = (p.M + most - 1) / most;; g++) {
    p.tokens = ((p.M + g - 1) / g + 15) / 16 * 16;
    p.groups = (p.M + p.tokens - 1) / p.tokens;      // (rounding up may leave nothing for the last one)
    tiles = ((long)p.N + per_tile - 1) / per_tile * p.groups;
    // the widest split whose clusters are all resident at once (of six CTAs 45 fit, not 49: a cluster stays within a part of the GPU)
    p.split = 1;
    for (int c = 2; c <= 8 && 2 * c <= p.kblocks; c++)
      if (tiles <= clusters[dev][c].load(std::memory_order_acquire)) p.split = c;
    sums = p.tokens * 512;
    lows = OP == kAdapt ? ((p.tokens * 32 + p.split - 1) / p.split + 1) * 16 : 0;
    if (sums + lows <= kBudget - 1024) break;        // 128 rows of one CTA with their low-rank parts are too many
  }
  if (tiles * p.split > 0x7fffffffL) return FP4AR_ERR_ARGUMENT;
  CUtensorMap mw, mx;
  if (!map_2d(&mw, w, rows, OP == kInput ? p.N : K, 64) || !map_2d(&mx, x, p.M, K, p.tokens)) return FP4AR_ERR_UNSUPPORTED;
  const int stage = kOpBytes + p.tokens * 128, blocks = (p.kblocks + p.split - 1) / p.split;
  p.stages = (kBudget - 1024 - lows) / stage;
  if (p.stages > kFewStagesMax) p.stages = kFewStagesMax;
  if (p.stages > blocks) p.stages = blocks;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(tiles * p.split));
  cfg.blockDim = dim3(kFewThreads<OP>);
  p.low_offset = p.stages * stage > sums ? p.stages * stage : sums;
  // Never so little that more CTAs fit an SM than its TMEM has columns for: one that waits for columns while its cluster waits for it, and
  // another the other way round, would wait for ever.
  const int least = (WIDE ? 116 : 78) * 1024, needed = p.low_offset + lows + 1024;
  cfg.dynamicSmemBytes = needed > least ? needed : least;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, few_rows_kernel<OP, WIDE>, mw, mx, p) != cudaSuccess) return cuda_fail();
  return cuda_check_launch();
}

}  // namespace layer
}  // namespace fp4ar
