// The row-parallel linear with low-rank adapters of many requests: y_i = x_i W^T + s_a (x_i A_a^T) B_a^T, a = ids[i].
//
// Two launches: a first kernel computes V[i] = s_a x_i A_a^T and lists the adapters of every 256 rows; the product with W then takes
// V_a B_a^T into the same accumulators (layer_gemm.cuh).
#include <algorithm>

#include "few_rows.cuh"
#include "layer_gemm.cuh"

namespace fp4ar {
namespace layer {

struct Workspace {
  __nv_bfloat16* v;      // [M][chunks][64]: V as layer_gemm.cuh takes it
  int* lists;            // [row tiles][kListStride]
  size_t bytes;
  Workspace(void* base, int M, int R) {
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    char* p = (char*)base;
    const size_t vb = up((size_t)M * ((R + kChunk - 1) / kChunk) * 128);
    v = (__nv_bfloat16*)p;
    lists = (int*)(p + vb);
    bytes = vb + up(((size_t)M + 255) / 256 * kListStride * 4);
  }
};

struct LowParams {
  int M, R, adapters, kblocks, split;
  const int* ids;
  const float* scales;
  __nv_bfloat16* v;
  int* lists;
  StatusWords* status;
  unsigned long long timeout_ns;
};

// V of 128 rows, the first launch.  x goes once through shared memory for all adapters of the rows: B of the product are the A_a of up to
// 256 / R of them, one behind the other (more adapters take more passes), every row is multiplied with all of them, and the
// epilogue keeps of each row the columns of its own adapter.  So what another adapter or row holds reaches nobody else, and the
// time is that of reading x.  A cluster of `split` CTAs cuts K where there are few rows; their sums meet in shared memory, in the
// order of the CTAs.
// The ring's stages are as large as the adapters of the rows need (8192 x 8192, rank 64: four stages for 256 rows of A 42 us, eight for one
// adapter 36, which is 151 MB at 4.2 TB/s, launch, lists and the exchange of the sums, about 5 us, included; 4096 x 2048, rank 16, two CTAs
// for 128 rows: 13 us.)
constexpr int kLowStagesMax = 10;
__host__ __device__ constexpr int low_ring(int R) { return (R <= 64 ? 4 : 3) * (kOpBytes + 256 * kBlockK * 2); }
__host__ __device__ constexpr int low_smem(int R) { return low_ring(R) + 128 * R * 4 + 1024; }

// Whether `id` is among the first `n` of sid.
__device__ __forceinline__ bool seen_before(const int* sid, int n, int id) {
  bool seen = false;
#pragma unroll 8
  for (int i = 0; i < n; i += 4) {
    const int4 s = *reinterpret_cast<const int4*>(sid + i);
    seen = seen | (s.x == id) | (s.y == id && i + 1 < n) | (s.z == id && i + 2 < n) | (s.w == id && i + 3 < n);
  }
  return seen;
}
__device__ __forceinline__ void rows_barrier() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }      // warps 2-5

__global__ void __launch_bounds__(192, 1)
low_rank_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ LowParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kLowStagesMax], empty[kLowStagesMax], acc_full, acc_empty;
  __shared__ uint32_t tmem_holder;
  __shared__ volatile uint32_t abort_flag;
  __shared__ __align__(16) int sid[256];
  __shared__ int list[128], wcount[4], scount[4], scount2[4], count;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* part = reinterpret_cast<float*>(ring + low_ring(p.R));            // [128][R]
  float* scale = reinterpret_cast<float*>(ring);                           // [128], behind the last product
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = blockIdx.x / p.split, crank = blockIdx.x % p.split, row0 = tile * 128;
  if (tid == 0) {
    for (int s = 0; s < kLowStagesMax; s++) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    mbar_init(&acc_full, 1);
    mbar_init(&acc_empty, 4);
    abort_flag = 0u;
    mbar_init_fence();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_a);
  }
  if (warp == 1) { tmem_alloc(&tmem_holder, 256); tmem_relinquish(); }
  GemmWait gw{&abort_flag, p.status, p.timeout_ns};
  pdl_wait_prior_grids();
  pdl_release_dependents();                              // after the wait: the product with W relies on it

  // the distinct adapters of the 128 rows, in the order of their first rows; thread 64 + r has row r
  auto id_of = [&](int row) {
    const int id = row < p.M ? p.ids[row] : -1;
    return id < p.adapters ? id : -1;
  };
  const int r = tid - 64;
  int id = -1;
  bool first = false;
  uint32_t votes = 0;
  int* const firsts = sid + 128;                         // those of each warp's rows; the list of 256 rows overwrites them later
  if (r >= 0) {
    sid[r] = id = id_of(row0 + r);
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    first = id >= 0 && lane == __ffs(same) - 1;
    votes = __ballot_sync(0xffffffffu, first);
    if (first) firsts[(warp - 2) * 32 + __popc(votes & ((1u << lane) - 1u))] = id;
    if (lane == 0) wcount[warp - 2] = __popc(votes);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (r >= 0) {
    for (int w = 0; w < warp - 2; w++)
      for (int i = 0; i < wcount[w]; i++) first = first && firsts[w * 32 + i] != id;
    votes = __ballot_sync(0xffffffffu, first);
    if (lane == 0) scount[warp - 2] = __popc(votes);
  }
  __syncthreads();
  if (first) {
    int at = __popc(votes & ((1u << lane) - 1u));
    for (int w = 0; w < warp - 2; w++) at += scount[w];
    list[at] = id;
  }
  if (tid == 64) count = scount[0] + scount[1] + scount[2] + scount[3];
  __syncthreads();
  const uint32_t tmem_base = tmem_holder;
  const int rp = (p.R + 15) / 16 * 16, group = 256 / rp, passes = (count + group - 1) / group;
  const int kb0 = p.kblocks * crank / p.split, kb1 = p.kblocks * (crank + 1) / p.split;
  const int stage_bytes = kOpBytes + min(group, count) * rp * 128, stages = min(low_ring(p.R) / stage_bytes, kLowStagesMax);
  int issued = 0;

  if (warp == 0) {
    if (lane == 0) {
      for (int ps = 0; ps < passes; ps++) {
        const int n = min(group, count - ps * group);
        for (int kb = kb0; kb < kb1; kb++, issued++) {
          const int s = issued % stages;
          if (!gemm_wait(empty + s, ((issued / stages) & 1u) ^ 1u, gw, 1)) goto done;
          uint8_t* at = ring + s * stage_bytes;
          mbar_arrive_expect(full + s, kOpBytes + n * rp * 128);
          tma_load_2d(at, &map_x, kb * kBlockK, row0, full + s);
          for (int i = 0; i < n; i++) tma_load_2d(at + kOpBytes + i * rp * 128, &map_a, kb * kBlockK, list[ps * group + i] * p.R, full + s);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int it = 0;
      for (int ps = 0; ps < passes; ps++) {
        const int n = min(group, count - ps * group) * rp;
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
        if (!gemm_wait(&acc_empty, (ps & 1u) ^ 1u, gw, 2)) goto done;
        tc_fence_after();
        for (int kb = kb0; kb < kb1; kb++, it++) {
          const int s = it % stages;
          if (!gemm_wait(full + s, (it / stages) & 1u, gw, 3)) goto done;
          tc_fence_after();
          const uint64_t da = umma_desc_k128(ring + s * stage_bytes), db = umma_desc_k128(ring + s * stage_bytes + kOpBytes);
#pragma unroll
          for (int k = 0; k < kBlockK / 16; k++) umma_bf16(tmem_base, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc, kb > kb0 || k ? 1u : 0u);
          umma_commit(empty + s);
        }
        umma_commit(&acc_full);
      }
    }
  } else {
    if ((tile & 1) == 0 && crank == 0) {
      // the list of 256 rows for the product with W: these 128 rows' and what the other 128 add
      sid[128 + r] = id = id_of(row0 + 128 + r);
      rows_barrier();
      const bool adds = id >= 0 && !seen_before(sid, 128 + r, id);
      votes = __ballot_sync(0xffffffffu, adds);
      if (lane == 0) scount2[warp - 2] = __popc(votes);
      rows_barrier();
      int* out = p.lists + (size_t)(tile >> 1) * kListStride;
      if (r < count) out[1 + r] = list[r];
      if (adds) {
        int at = count + __popc(votes & ((1u << lane) - 1u));
        for (int w = 0; w < warp - 2; w++) at += scount2[w];
        out[1 + at] = id;
      }
      if (r == 0) out[0] = count + scount2[0] + scount2[1] + scount2[2] + scount2[3];
    }
    // TMEM lane quarter warp & 3 has rows 32 (warp & 3) ...
    const int q = warp & 3, row = q * 32 + lane;
    const int mine = sid[row];
    const float factor = mine >= 0 && p.scales ? p.scales[mine] : 1.0f;
    for (int ps = 0; ps < passes; ps++) {
      if (!__all_sync(0xffffffffu, gemm_wait(&acc_full, ps & 1u, gw, 4))) break;
      tc_fence_after();
      const int n = min(group, count - ps * group);
      for (int i = 0; i < n; i++) {
        const bool take = mine == list[ps * group + i];
        if (!__any_sync(0xffffffffu, take)) continue;
        for (int c = 0; c < rp; c += 32) {               // beyond rp: columns of the next adapter or unused ones (256 + 16 are never reached: rp = 16 then)
          float v[32];
          const uint32_t at = tmem_base + ((uint32_t)(q * 32) << 16) + i * rp + c;
          const int cols = min(32, rp - c);
          if (cols == 32) tmem_ld32_issue(at, v); else tmem_ld16_issue(at, v);
          tmem_ld_wait();
          if (take) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (c + e < p.R) *reinterpret_cast<float4*>(part + row * p.R + c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty);
    }
    scale[row] = factor;                                 // the last product is through with the ring
  }
done:
  tc_fence_before();
  __syncthreads();
  if (abort_flag != 0u) {
    if (tid == 0)
      for (int i = max(0, issued - stages); i < issued; i++) gemm_settle(full + i % stages, (i / stages) & 1);
    if (tid == 32) {
      __shared__ uint64_t settled;
      mbar_init(&settled, 1);
      umma_commit(&settled);
      gemm_settle(&settled, 0u);
    }
    __syncthreads();
  }
  if (p.split > 1) cluster_sync_all();
  // this CTA's share of the rows: the sum of the cluster's parts, scaled, as two BF16 halves; four columns of a row per thread
  const int share = 128 / p.split, padded = (p.R + kChunk - 1) / kChunk * kChunk, per_row = padded / 4, rows = 32 / per_row;
  const int n = lane % per_row * 4;
  for (int i = warp * rows + lane / per_row; i < share && lane < rows * per_row; i += 6 * rows) {
    const int rr = crank * share + i;
    if (sid[rr] < 0) continue;                           // nobody reads its V
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (n < p.R) {
      if (p.split == 1) {
        s = *reinterpret_cast<const float4*>(part + rr * p.R + n);
      } else {
        float4 f[8];                                     // all of them in flight
#pragma unroll
        for (int d = 0; d < 8; d++)
          if (d < p.split) f[d] = cluster_ld4(cluster_addr(part + rr * p.R + n, d));
#pragma unroll
        for (int d = 0; d < 8; d++)
          if (d < p.split) { s.x += f[d].x; s.y += f[d].y; s.z += f[d].z; s.w += f[d].w; }
      }
      const float sc = scale[rr];
      s.x *= sc; s.y *= sc; s.z *= sc; s.w *= sc;
    }
    // the rounded value and what the rounding left; what is not finite stays in the first alone
    auto left = [](float v, float rounded) { const float l = v - rounded; return fabsf(l) <= 3.4e38f ? l : 0.0f; };
    const uint2 hi = make_uint2(pack_bf16(s.x, s.y), pack_bf16(s.z, s.w));
    __nv_bfloat16* line = p.v + (size_t)(row0 + rr) * (2 * padded) + n / kChunk * 64 + n % kChunk;
    *reinterpret_cast<uint2*>(line) = hi;
    *reinterpret_cast<uint2*>(line + kChunk) = make_uint2(pack_bf16(left(s.x, bf16_lo(hi.x)), left(s.y, bf16_hi(hi.x))),
                                                          pack_bf16(left(s.z, bf16_lo(hi.y)), left(s.w, bf16_hi(hi.y))));
  }
  if (p.split > 1) cluster_sync_relaxed();               // a CTA's part is read until here
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

static int launch_low_rank(const void* x, const void* a, int K, LowParams p, cudaStream_t stream) {
  static std::atomic<int> raised[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cuda_fail();
  if (!raised[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(low_rank_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, low_smem(64) > low_smem(128) ? low_smem(64) : low_smem(128)) != cudaSuccess)
      return cuda_fail();
    raised[dev].store(1, std::memory_order_release);
  }
  p.status = gemm_status_word();
  if (!p.status) return cuda_fail();
  p.timeout_ns = kWaitLimitNs;
  CUtensorMap mx, ma;
  if (!map_2d(&mx, x, p.M, K, 128) || !map_2d(&ma, a, (long)p.adapters * p.R, K, (p.R + 15) / 16 * 16)) return FP4AR_ERR_UNSUPPORTED;
  // Up to eight CTAs per 128 rows.  Where a quarter of the SMs will do, no more: the product with W starts on the others meanwhile, and there
  // V is to be ready when its first tiles are.  But two at least, since one takes longer than the tile (4096 x 2048 rows, N = 6144, all:
  // 105 us with one, 98.5 with two; 1031 x 1992 with 36 CTAs 41, with 72 or 144 43.5).
  const int tiles = (p.M + 127) / 128, sms = device_sm_count(), most = 4 * tiles <= sms ? std::max(sms / 4, 2 * tiles) : sms;
  p.split = 1;
  while (p.split < 8 && 2 * p.split * tiles <= most && 2 * p.split <= p.kblocks) p.split *= 2;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(tiles * p.split);
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = low_smem(p.R);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, low_rank_kernel, mx, ma, p) != cudaSuccess) return cuda_fail();
  return cuda_check_launch();
}

__device__ __forceinline__ uint4 ldg16(const uint4* p) {      // volatile: issued in the order written, ahead of the arithmetic
  uint4 r;
  asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// V of few rows: eight ranks of a row per CTA, a warp for each, eight loads of every lane of x and of A_a in flight.  Bound by latency: 64 rows
// of 48 adapters, K = 2048, rank 16: 4.6 us alone, of which 2.4 are those of a launch that finds no adapters; K = 8192, rank 64: 15 us.
__global__ void __launch_bounds__(256, 3) few_low_rank_kernel(const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ a,
                                                           const int* __restrict__ ids, const float* __restrict__ scales, int K, int R, int adapters,
                                                           __nv_bfloat16* __restrict__ v) {
  pdl_wait_prior_grids();
  pdl_release_dependents();                              // after the wait: the product with W relies on it
  const int row = blockIdx.x, r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int id = ids[row];
  if (id < 0 || id >= adapters) return;                  // nobody reads its V
  const uint4* xp = reinterpret_cast<const uint4*>(x + (size_t)row * K);
  const uint4* ap = reinterpret_cast<const uint4*>(a + ((size_t)id * R + r) * K);
  float s = 0.0f;
  for (int i = lane; i < K / 8; i += 256) {
    uint4 xv[8], av[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int at = min(i + 32 * j, K / 8 - 1);
      av[j] = ldg16(ap + at);
      xv[j] = ldg16(xp + at);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (i + 32 * j >= K / 8) xv[j] = make_uint4(0, 0, 0, 0), av[j] = make_uint4(0, 0, 0, 0);
      const uint32_t xw[4] = {xv[j].x, xv[j].y, xv[j].z, xv[j].w}, aw[4] = {av[j].x, av[j].y, av[j].z, av[j].w};
#pragma unroll
      for (int e = 0; e < 4; e++) s = fmaf(bf16_hi(xw[e]), bf16_hi(aw[e]), fmaf(bf16_lo(xw[e]), bf16_lo(aw[e]), s));
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) {
    if (scales) s *= scales[id];
    const __nv_bfloat16 hi = __float2bfloat16_rn(s);
    const float left = s - __bfloat162float(hi);
    __nv_bfloat16* line = v + ((size_t)row * ((R + kChunk - 1) / kChunk) + r / kChunk) * 64 + r % kChunk;
    line[0] = hi;
    line[kChunk] = __float2bfloat16_rn(fabsf(left) <= 3.4e38f ? left : 0.0f);
  }
}

// Which of the two products takes a call.  For every adapter in a tile of 256 rows a call in tiles pays about 1.5 us at rank 16, K = 2048, and
// 5 - 6 at rank 64, K = 8192 (V's passes over x among them), the few-row kernel next to nothing, but it reads W once for every 128 rows
// and B once for every row.  N = 6144, us, few-row kernel / tiles.  K = 2048, rank 16: 200 rows of 4 adapters 24 / 22, of 8: 25 / 27, of 12: 25 / 33; 300 rows of 8: 28 / 27, of 12: 28 / 33,
// of 18: 28 / 43; 512 rows of 8: 38 / 27, of 16: 38 / 39, of 20: 38 / 47, of 31: 38 / 62, of 64: 37 / 130.  K = 8192, rank 64: 256 rows of
// 8: 95 / 77, of 15: 96 / 116, of 64: 103 / 427; 512 rows of 16: 158 / 106, of 31: 158 / 183.
// The limit of M / 16 adapters is thus too high, by up to twice at rank 16 (the two cross at 7 of 200, 9 of 300 and 15 of 512 rows), by a
// fifth to a half at rank 64 (11 of 256, 26 of 512): just below it a call takes up to 1.6 times the other kernel's time.  How many
// adapters a tile has is known on the device alone, so the pool's size stands in for it.  Beyond 512 rows only tiles take a call: 1024
// rows of 1, 8 and 64 adapters 30, 48 and 198 us at rank 16, 35, 71 and 443 at rank 64 (K = 2048); 4096 rows 85, 129, 506 and 94, 176, 1113.
static bool few_rows(int M, int adapters) { return M <= kNarrowRows || (M <= 512 && 16LL * adapters >= M); }

}  // namespace layer
}  // namespace fp4ar

using namespace fp4ar;
using namespace fp4ar::layer;

static bool adapters_shape_ok(int M, int N, int K, int R, int adapters) {
  return M >= 0 && N >= 8 && K >= 8 && R >= 8 && R <= 128 && adapters >= 1 && N % 8 == 0 && K % 8 == 0 && R % 8 == 0 &&
         extents_ok((long long)M + 256, (long long)N + 256) && extents_ok((long long)adapters * N + 256, (long long)adapters * R + 256) && extents_ok((long long)M + 1024, adapters) &&
         extents_ok(K, 0);
}

extern "C" size_t fp4ar_adapters_workspace(int M, int R, int adapters) {
  if (M < 0 || R < 1 || adapters < 1) return 0;
  return Workspace(nullptr, M, R).bytes;
}

extern "C" int fp4ar_adapters_few_rows(int M, int adapters) {
  if (M < 0 || adapters < 1) return -1;
  return few_rows(M, adapters) ? 1 : 0;
}

extern "C" int fp4ar_linear_adapters(const void* x, const void* wt, const int* ids, const void* a, const void* b, const float* scales, int M,
                                     int N, int K, int R, int adapters, void* workspace, void* y, fp4ar_stream stream_) {
  if (!adapters_shape_ok(M, N, K, R, adapters)) return FP4AR_ERR_ARGUMENT;
  if (M == 0) return FP4AR_OK;
  if (!x || !wt || !ids || !a || !b || !workspace || !y || !aligned16(x, wt, a, b) || !aligned16(workspace, y) || ((uintptr_t)ids & 3) ||
      ((uintptr_t)scales & 3))
    return FP4AR_ERR_ARGUMENT;
  const cudaStream_t stream = (cudaStream_t)stream_;
  const Workspace ws(workspace, M, R);
  if (few_rows(M, adapters)) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(M, R / 8);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, few_low_rank_kernel, (const __nv_bfloat16*)x, (const __nv_bfloat16*)a, ids, scales, K, R, adapters, ws.v) != cudaSuccess)
      return cuda_fail();
    FewParams fp;
    memset(&fp, 0, sizeof(fp));
    fp.M = M; fp.N = N; fp.out = (__nv_bfloat16*)y;
    fp.R = R; fp.adapters = adapters; fp.ids = ids; fp.v = ws.v; fp.b = (const __nv_bfloat16*)b;
    return launch_few_rows<kAdapt, false>(wt, N, x, K, fp, stream);
  }
  LowParams lp;
  memset(&lp, 0, sizeof(lp));
  lp.M = M; lp.R = R; lp.adapters = adapters; lp.kblocks = (K + 63) / 64;
  lp.ids = ids; lp.scales = scales; lp.v = ws.v; lp.lists = ws.lists;
  const int rc = launch_low_rank(x, a, K, lp, stream);
  if (rc != FP4AR_OK) return rc;
  Maps maps;
  memset(&maps, 0, sizeof(maps));
  if (!map_2d(&maps.a, x, M, K, 128) || !map_2d(&maps.b, wt, N, K, 128) || !map_2d(&maps.out, y, M, N, 32) ||
      !map_2d(&maps.low, b, (long)adapters * N, R, 128))
    return FP4AR_ERR_UNSUPPORTED;
  Params p;
  memset(&p, 0, sizeof(p));
  p.M = M; p.N = N; p.kblocks = (K + 63) / 64;
  p.R = R; p.adapters = adapters; p.ids = ids; p.v = ws.v; p.lists = ws.lists; p.b = (const __nv_bfloat16*)b;
  return launch_pair_gemm<kAdapt>(maps, p, stream);
}
