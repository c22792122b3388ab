// The row-parallel linear with low-rank adapters of many requests: y_i = x_i W^T + s_a (x_i A_a^T) B_a^T, a = ids[i].
//
// Two launches: a first kernel computes V[i] = s_a x_i A_a^T, lists the adapters of every 256 rows and looks for infinities and NaN in
// the B of the adapters in use; the product with W then takes V_a B_a^T into the same accumulators (layer_gemm.cuh).
#include "layer_gemm.cuh"

namespace fp4ar {
namespace layer {

struct Workspace {
  float* v;              // [M][R]
  int* lists;            // [row tiles][kListStride]
  unsigned char* unsafe; // [adapters]
  size_t bytes;
  Workspace(void* base, int M, int R, int adapters) {
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    char* p = (char*)base;
    const size_t vb = up((size_t)M * R * 4), lb = up(((size_t)M + 255) / 256 * kListStride * 4);
    v = (float*)p;
    lists = (int*)(p + vb);
    unsafe = (unsigned char*)(p + vb + lb);
    bytes = vb + lb + up((size_t)adapters);
  }
};

struct LowParams {
  const __nv_bfloat16 *x, *a, *b;
  const int* ids;
  const float* scales;
  int M, N, K, R, adapters, row_ctas, list_ctas;
  float* v;
  int* lists;
  unsigned char* unsafe;
};

// Blocks 0 .. row_ctas-1: one row each; then one block per 256 rows for the lists; then one block per adapter for its check.
__global__ void __launch_bounds__(256) low_rank_kernel(const __grid_constant__ LowParams p) {
  __shared__ int sid[256];
  __shared__ int total;
  pdl_wait_prior_grids();
  pdl_release_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int block = blockIdx.x;
  if (block < p.row_ctas) {
    const int id = p.ids[block];
    if (id < 0 || id >= p.adapters) return;              // nobody reads its V
    const float scale = p.scales ? p.scales[id] : 1.0f;
    const uint4* x = reinterpret_cast<const uint4*>(p.x + (size_t)block * p.K);
    for (int r = warp; r < p.R; r += 8) {
      const uint4* a = reinterpret_cast<const uint4*>(p.a + ((size_t)id * p.R + r) * p.K);
      float s = 0.0f;
      for (int i = lane; i < p.K / 8; i += 32) {
        const uint4 xv = x[i], av = a[i];
        const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w}, aw[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
        for (int e = 0; e < 4; e++) s = fmaf(bf16_hi(xw[e]), bf16_hi(aw[e]), fmaf(bf16_lo(xw[e]), bf16_lo(aw[e]), s));
      }
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) p.v[(size_t)block * p.R + r] = s * scale;
    }
    return;
  }
  block -= p.row_ctas;
  if (block < p.list_ctas) {
    // the distinct adapters of 256 rows in the order of their first rows
    const int row = block * 256 + tid;
    int id = row < p.M ? p.ids[row] : -1;
    if (id >= p.adapters) id = -1;
    sid[tid] = id;
    if (tid == 0) total = 0;
    __syncthreads();
    bool first = id >= 0;
    for (int s = 0; s < tid; s++) first = first && sid[s] != id;
    __syncthreads();
    int before = 0;
    sid[tid] = first;
    __syncthreads();
    for (int s = 0; s < tid; s++) before += sid[s];
    int* list = p.lists + (size_t)block * kListStride;
    if (first) { list[1 + before] = id; atomicAdd(&total, 1); }
    __syncthreads();
    if (tid == 0) list[0] = total;
    return;
  }
  block -= p.list_ctas;
  if (tid == 0) total = 0;
  __syncthreads();
  bool used = false;
  for (int i = tid; i < p.M; i += 256) used = used || p.ids[i] == block;
  bool bad = false;
  if (__syncthreads_or(used)) {
    const uint4* b = reinterpret_cast<const uint4*>(p.b + (size_t)block * p.N * p.R);
    const size_t n = (size_t)p.N * p.R / 8;
    for (size_t i = tid; i < n; i += 256) {
      const uint4 w = b[i];
      for (uint32_t e : {w.x, w.y, w.z, w.w}) bad = bad || (e & 0x7F80u) == 0x7F80u || (e & 0x7F800000u) == 0x7F800000u;
    }
  }
  bad = __syncthreads_or(bad);
  if (tid == 0) p.unsafe[block] = bad;
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
  return Workspace(nullptr, M, R, adapters).bytes;
}

extern "C" int fp4ar_linear_adapters(const void* x, const void* wt, const int* ids, const void* a, const void* b, const float* scales, int M,
                                     int N, int K, int R, int adapters, void* workspace, void* y, fp4ar_stream stream_) {
  if (!adapters_shape_ok(M, N, K, R, adapters)) return FP4AR_ERR_ARGUMENT;
  if (M == 0) return FP4AR_OK;
  if (!x || !wt || !ids || !a || !b || !workspace || !y || !aligned16(x, wt, a, b) || !aligned16(workspace, y) || ((uintptr_t)ids & 3) ||
      ((uintptr_t)scales & 3))
    return FP4AR_ERR_ARGUMENT;
  const cudaStream_t stream = (cudaStream_t)stream_;
  const Workspace ws(workspace, M, R, adapters);
  LowParams lp{(const __nv_bfloat16*)x, (const __nv_bfloat16*)a, (const __nv_bfloat16*)b, ids, scales, M, N, K, R, adapters, M, (M + 255) / 256,
               ws.v, ws.lists, ws.unsafe};
  int rc = launch_dependent(low_rank_kernel, lp.row_ctas + lp.list_ctas + adapters, 256, stream, lp);
  if (rc != FP4AR_OK) return rc;
  Maps maps;
  memset(&maps, 0, sizeof(maps));
  if (!map_2d(&maps.a, x, M, K, 128) || !map_2d(&maps.b, wt, N, K, 128) || !map_2d(&maps.out, y, M, N, 32) ||
      !map_2d(&maps.low, b, (long)adapters * N, R, 128))
    return FP4AR_ERR_UNSUPPORTED;
  Params p;
  memset(&p, 0, sizeof(p));
  p.M = M; p.N = N; p.kblocks = (K + 63) / 64;
  p.R = R; p.adapters = adapters; p.ids = ids; p.v = ws.v; p.lists = ws.lists; p.unsafe = ws.unsafe; p.b = (const __nv_bfloat16*)b;
  return launch_pair_gemm<kAdapt>(maps, p, stream);
}
