// The row-parallel linear with low-rank adapters of many requests: y_i = x_i W^T + s_a (x_i A_a^T) B_a^T, a = ids[i].
//
// Two launches: a first kernel computes V[i] = s_a x_i A_a^T and lists the adapters of every 256 rows; the product with W then takes
// V_a B_a^T into the same accumulators (layer_gemm.cuh).
#include <cooperative_groups.h>
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
  const __nv_bfloat16 *x, *a;
  const int* ids;
  const float* scales;
  int M, K, R, adapters, split;
  __nv_bfloat16* v;
  int* lists;
};

__device__ __forceinline__ void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// The distinct adapters of 256 rows in the order of their first rows, by 256 threads.
__device__ void list_adapters(const LowParams& p, int tile, int* sid, int* scount) {
  const int tid = threadIdx.x, row = tile * 256 + tid;
  int id = row < p.M ? p.ids[row] : -1;
  if (id >= p.adapters) id = -1;
  sid[tid] = id;
  __syncthreads();
  bool first = id >= 0;
  for (int s = 0; s < tid; s++) first = first && sid[s] != id;
  const uint32_t votes = __ballot_sync(0xffffffffu, first);
  if ((tid & 31) == 0) scount[tid >> 5] = __popc(votes);
  __syncthreads();
  int before = __popc(votes & ((1u << (tid & 31)) - 1u)), total = 0;
  for (int w = 0; w < 8; w++) {
    if (w < tid >> 5) before += scount[w];
    total += scount[w];
  }
  int* list = p.lists + (size_t)tile * kListStride;
  if (first) list[1 + before] = id;
  if (tid == 0) list[0] = total;
}

// V of 64 rows x 8 NT ranks: a cluster of `split` CTAs cuts K, the eight warps of a CTA cut its share, and the sums meet in shared
// memory, warps first, CTAs next, always in the same order.
//
// A warp takes 32 K columns at a time.  Operands go from global memory to registers without a stop: a lane's 16 bytes of a row are
// columns 8 t .. 8 t + 7 of the 32 (t = lane & 3), and since x and A use the same columns, their order inside the product does
// not matter: words 0, 1 are one mma.sync m16n8k16, words 2, 3 the next.  (tcgen05 has nothing to give here: the product has a
// third of the operations per byte that would make it matter, and a tile of x would have to go through shared memory for every
// adapter in it.)  x of the next 32 columns is in flight during the products.
// Rows of a tile with several adapters: one pass for each, over the groups of 16 rows that have it, and of its results only those
// rows are kept, so what another adapter holds reaches nobody else.
// Bound by the reads of x: ...
template <int NT>
__global__ void __launch_bounds__(256, 1) low_rank_kernel(const __grid_constant__ LowParams p) {
  constexpr int kCols = 8 * NT;
  extern __shared__ float red[];                        // [8 warps][64 rows][kCols], then the CTA's sums [64][kCols]
  __shared__ int sid[256];
  __shared__ int scount[8];
  float* part = red + 8 * 64 * kCols;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 2, t = lane & 3;
  const int tile = blockIdx.x / p.split, crank = blockIdx.x % p.split, row0 = tile * 64;
  pdl_wait_prior_grids();
  pdl_release_dependents();
  if ((tile & 3) == 0 && crank == 0) list_adapters(p, tile >> 2, sid, scount);

  // both halves of the tile's ids
  int id0 = row0 + lane < p.M ? p.ids[row0 + lane] : -1, id1 = row0 + 32 + lane < p.M ? p.ids[row0 + 32 + lane] : -1;
  if (id0 < 0 || id0 >= p.adapters) id0 = -1;
  if (id1 < 0 || id1 >= p.adapters) id1 = -1;
  const unsigned long long have = ((unsigned long long)__ballot_sync(0xffffffffu, id1 >= 0) << 32) | __ballot_sync(0xffffffffu, id0 >= 0);
  const int chunks = (p.K + 31) / 32, step = 8 * p.split;

  for (int r0 = 0; r0 < p.R; r0 += kCols) {
    for (unsigned long long left = have; left;) {
      const int f = __ffsll((long long)left) - 1;
      const int adapter = __shfl_sync(0xffffffffu, f < 32 ? id0 : id1, f & 31);
      const unsigned long long rows = ((unsigned long long)__ballot_sync(0xffffffffu, id1 == adapter) << 32) | __ballot_sync(0xffffffffu, id0 == adapter);
      left &= ~rows;
      float acc[4][NT][4];
#pragma unroll
      for (int m = 0; m < 4; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.0f;
      const __nv_bfloat16* a = p.a + (size_t)adapter * p.R * p.K;
      auto x_word = [&](int m, int half, int k) {        // 8 columns of row 16 m + 8 half + grp
        const int row = row0 + 16 * m + 8 * half + grp;
        return (rows >> (16 * m) & 0xFFFFull) && row < p.M && k < p.K ? ldg16(p.x + (size_t)row * p.K + k) : make_uint4(0, 0, 0, 0);
      };
      int c = crank * 8 + warp;
      uint4 xs[4][2];
      if (c < chunks) {
#pragma unroll
        for (int m = 0; m < 4; m++) { xs[m][0] = x_word(m, 0, c * 32 + 8 * t); xs[m][1] = x_word(m, 1, c * 32 + 8 * t); }
      }
      for (; c < chunks; c += step) {
        const int k = c * 32 + 8 * t, next = k + 32 * step;
        uint4 as[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const int r = r0 + 8 * n + grp;
          as[n] = r < p.R && k < p.K ? __ldg(reinterpret_cast<const uint4*>(a + (size_t)r * p.K + k)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int m = 0; m < 4; m++) {
          const uint4 x0 = xs[m][0], x1 = xs[m][1];
          xs[m][0] = x_word(m, 0, next);
          xs[m][1] = x_word(m, 1, next);
          if (rows >> (16 * m) & 0xFFFFull) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
              mma_bf16(acc[m][n], x0.x, x1.x, x0.y, x1.y, as[n].x, as[n].y);
              mma_bf16(acc[m][n], x0.z, x1.z, x0.w, x1.w, as[n].z, as[n].w);
            }
          }
        }
      }
      // rows 16 m + grp and + 8 of this adapter, columns 8 n + 2 t, + 1
#pragma unroll
      for (int m = 0; m < 4; m++)
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const int r = 16 * m + 8 * half + grp;
          if (rows >> r & 1ull) {
#pragma unroll
            for (int n = 0; n < NT; n++)
              *reinterpret_cast<float2*>(red + (warp * 64 + r) * kCols + 8 * n + 2 * t) = make_float2(acc[m][n][2 * half], acc[m][n][2 * half + 1]);
          }
        }
    }
    __syncthreads();
    for (int i = tid; i < 64 * kCols; i += 256) {
      float s = 0.0f;
      if (have >> (i / kCols) & 1ull) {
#pragma unroll
        for (int w = 0; w < 8; w++) s += red[w * 64 * kCols + i];
      }
      part[i] = s;
    }
    if (p.split > 1) cooperative_groups::this_cluster().sync(); else __syncthreads();
    const int share = 64 / p.split, padded = (p.R + kChunk - 1) / kChunk * kChunk;
    for (int i = tid; i < share * kCols; i += 256) {
      const int r = crank * share + i / kCols, n = i % kCols;
      if (!(have >> r & 1ull) || r0 + n >= padded) continue;
      float s = 0.0f;
      for (int d = 0; d < p.split; d++) {
        const float* from = p.split > 1 ? cooperative_groups::this_cluster().map_shared_rank(part, d) : part;
        s += from[r * kCols + n];
      }
      if (p.scales) s *= p.scales[p.ids[row0 + r]];
      // the rounded value and what the rounding left; what is not finite stays in the first alone
      const __nv_bfloat16 hi = __float2bfloat16_rn(s);
      const float left = s - __bfloat162float(hi);
      __nv_bfloat16* line = p.v + (size_t)(row0 + r) * (2 * padded) + (r0 + n) / kChunk * 64 + n % kChunk;
      line[0] = hi;
      line[kChunk] = __float2bfloat16_rn(fabsf(left) <= 3.4e38f ? left : 0.0f);
    }
    if (p.split > 1) cooperative_groups::this_cluster().sync(); else __syncthreads();
  }
}

template <int NT>
static int launch_low_rank(LowParams p, cudaStream_t stream) {
  constexpr int kBytes = 9 * 64 * 8 * NT * 4;
  static std::atomic<int> raised[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cuda_fail();
  if (!raised[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(low_rank_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess) return cuda_fail();
    raised[dev].store(1, std::memory_order_release);
  }
  // as many CTAs per 64 rows, up to eight, as the SMs have room for
  const int tiles = (p.M + 63) / 64, sms = device_sm_count(), chunks = (p.K + 31) / 32;
  p.split = 1;
  while (p.split < 8 && 2 * p.split * tiles <= sms && 16 * p.split <= chunks) p.split *= 2;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(tiles * p.split);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, low_rank_kernel<NT>, p) != cudaSuccess) return cuda_fail();
  return cuda_check_launch();
}

}  // namespace layer
}  // namespace fp4ar

using namespace fp4ar;
using namespace fp4ar::layer;

static bool adapters_shape_ok(int M, int N, int K, int R, int adapters) {
  return M >= 0 && N >= 8 && K >= 8 && R >= 8 && R <= 128 && adapters >= 1 && N % 8 == 0 && K % 8 == 0 && R % 8 == 0 &&
         extents_ok((long long)M + 256, (long long)N + 256) && extents_ok((long long)adapters * N + 256, (long long)M + adapters + 1024) &&
         extents_ok(K, 0);
}

extern "C" size_t fp4ar_adapters_workspace(int M, int R, int adapters) {
  if (M < 0 || R < 1 || adapters < 1) return 0;
  return Workspace(nullptr, M, R).bytes;
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
  const LowParams lp{(const __nv_bfloat16*)x, (const __nv_bfloat16*)a, ids, scales, M, K, R, adapters, 1, ws.v, ws.lists};
  const int rc = R <= 16 ? launch_low_rank<2>(lp, stream) : R <= 32 ? launch_low_rank<4>(lp, stream) : launch_low_rank<8>(lp, stream);
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
