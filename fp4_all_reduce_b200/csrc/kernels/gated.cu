// Gated projections of the feed-forward block: h = a(x Wg^T) * (x Wu^T) in one kernel (layer_gemm.cuh), and their gradients.
//
// Backward: dpre = (dh u a'(g), dh a(g)) elementwise from the projections that the forward pass kept, then two products dx = dpre W
// and dW = dpre^T x.  The projections are kept in FP32: in BF16 their rounding doubles the gradients' error (relative to
// 64 bits 0.0030 instead of 0.0024, where the rounding of the results alone is 0.0017).  dpre is rounded to BF16, the type that
// the tensor cores take.
#include "few_rows.cuh"
#include "layer_gemm.cuh"

namespace fp4ar {
namespace layer {

// One thread has eight neighbouring columns of a row: five 16-byte loads, two 16-byte stores, 14 bytes for each column of dh.
// Bound by memory: 4096 x 2048, 117 MB in 17.9 us alone, 6.6 TB/s; 2048 x 2048 in 10.
template <int ACT>
__global__ void gated_grad_kernel(const uint4* __restrict__ dh, const float4* __restrict__ pre, uint4* __restrict__ dpre, int M, int f8) {
  pdl_wait_prior_grids();
  pdl_release_dependents();
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= f8) return;
  for (long row = blockIdx.y; row < M; row += gridDim.y) {
    const uint4 d = dh[row * f8 + c];
    const float4 *gp = pre + (row * 2 * f8 + c) * 2, *up = gp + 2L * f8;
    const float4 g[2] = {gp[0], gp[1]}, u[2] = {up[0], up[1]};
    const uint32_t dw[4] = {d.x, d.y, d.z, d.w};
    uint32_t og[4], ou[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float4 &g4 = g[i >> 1], &u4 = u[i >> 1];
      float a0, s0, a1, s1;
      act_both<ACT>(i & 1 ? g4.z : g4.x, a0, s0);
      act_both<ACT>(i & 1 ? g4.w : g4.y, a1, s1);
      const float d0 = bf16_lo(dw[i]), d1 = bf16_hi(dw[i]);
      og[i] = pack_bf16(d0 * (i & 1 ? u4.z : u4.x) * s0, d1 * (i & 1 ? u4.w : u4.y) * s1);
      ou[i] = pack_bf16(d0 * a0, d1 * a1);
    }
    dpre[row * 2 * f8 + c] = make_uint4(og[0], og[1], og[2], og[3]);
    dpre[(row * 2 + 1) * f8 + c] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
}

static int launch_grad(const void* dh, const void* pre, void* dpre, int M, int F, int act, cudaStream_t stream) {
  const int f8 = F / 8;
  const int block = f8 < 256 ? (f8 + 31) / 32 * 32 : 256, gx = (f8 + block - 1) / block;
  int gy = device_sm_count() * 16 * (256 / block) / gx;        // enough warps for every SM, then a walk over the rows
  gy = gy < 1 ? 1 : gy > M ? M : gy;
  if (gy > 65535) gy = 65535;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(gx, gy);
  cfg.blockDim = dim3(block);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = act == FP4AR_ACT_SILU ? gated_grad_kernel<FP4AR_ACT_SILU>
                : act == FP4AR_ACT_GELU ? gated_grad_kernel<FP4AR_ACT_GELU> : gated_grad_kernel<FP4AR_ACT_GELU_TANH>;
  if (cudaLaunchKernelEx(&cfg, kernel, (const uint4*)dh, (const float4*)pre, (uint4*)dpre, M, f8) != cudaSuccess) return cuda_fail();
  return cuda_check_launch();
}

// Which kernel takes a product of M rows whose output has `cols` columns, `per_tile` of them to a tile of 256 rows: up to 128 rows the one
// for few rows, and up to 1024 where the other would keep no more than a third of the units busy.  us, few-row kernel / tiles, forward:
// K = 6144, F = 2048: 200 rows (16 tiles) 20 / 29, 333 (32 tiles) 30 / 32, 512 (32) 34 / 33; F = 8192: 200 rows (64) 51 / 44.  dx of K = 2048, F = 2056:
// 512 rows (16 tiles) 22 / 30, 640 (24) 29 / 30, 1024 (32) 32 / 30; of K = 6144, F = 2048: 256 rows (24) 28 / 27, 333 (48) 36 / 29.
static bool few_rows(int M, int cols, int per_tile) {
  if (M <= kNarrowRows) return true;
  const long tiles = (M + 255L) / 256 * ((cols + per_tile - 1L) / per_tile);
  return M <= 1024 && 3 * tiles <= device_sm_count() / 2;
}

static bool shape_ok(int M, int F, int K, int act) {
  return M >= 0 && F >= 8 && K >= 8 && F % 8 == 0 && K % 8 == 0 && act >= FP4AR_ACT_SILU && act <= FP4AR_ACT_GELU_TANH &&
         extents_ok((long long)M + 256, 2LL * F + 256) && extents_ok(K, 0);
}

}  // namespace layer
}  // namespace fp4ar

using namespace fp4ar;
using namespace fp4ar::layer;

extern "C" int fp4ar_gated_linear(const void* x, const void* wt, int M, int F, int K, int act, void* h, void* pre, fp4ar_stream stream) {
  if (!shape_ok(M, F, K, act)) return FP4AR_ERR_ARGUMENT;
  if (M == 0) return FP4AR_OK;
  if (!x || !wt || !h || !aligned16(x, wt, h, pre)) return FP4AR_ERR_ARGUMENT;
  if (few_rows(M, F, 128)) {
    FewParams fp;
    memset(&fp, 0, sizeof(fp));
    fp.M = M; fp.N = F; fp.act = act; fp.out = (__nv_bfloat16*)h; fp.pre = (float*)pre;
    return M <= kNarrowRows ? launch_few_rows<kGated, false>(wt, 2L * F, x, K, fp, (cudaStream_t)stream)
                            : launch_few_rows<kGated, true>(wt, 2L * F, x, K, fp, (cudaStream_t)stream);
  }
  Maps maps;
  memset(&maps, 0, sizeof(maps));
  if (!map_2d(&maps.a, x, M, K, 128) || !map_2d(&maps.b, wt, 2L * F, K, 128) || !map_2d(&maps.out, h, M, F, 32) ||
      (pre && !map_pre(&maps.pre, pre, M, F)))
    return FP4AR_ERR_UNSUPPORTED;
  Params p;
  memset(&p, 0, sizeof(p));
  p.M = M; p.N = F; p.kblocks = (K + 63) / 64; p.act = act; p.want_pre = pre != nullptr;
  return launch_pair_gemm<kGated>(maps, p, (cudaStream_t)stream);
}

extern "C" int fp4ar_gated_backward(const void* dh, const void* pre, const void* x, const void* wt, int M, int F, int K, int act,
                                    void* dpre, void* dx, void* dwt, fp4ar_stream stream_) {
  if (!shape_ok(M, F, K, act)) return FP4AR_ERR_ARGUMENT;
  const cudaStream_t stream = (cudaStream_t)stream_;
  if (M == 0) {
    if (dwt && cudaMemsetAsync(dwt, 0, (size_t)2 * F * K * 2, stream) != cudaSuccess) return cuda_fail();
    return FP4AR_OK;
  }
  if (!dh || !pre || !dpre || (dx && !wt) || (dwt && !x) || !aligned16(dh, pre, dpre) || !aligned16(x, wt, dx, dwt)) return FP4AR_ERR_ARGUMENT;
  int rc = launch_grad(dh, pre, dpre, M, F, act, stream);
  if (rc != FP4AR_OK) return rc;
  Params p;
  if (dx && few_rows(M, K, 256)) {
    FewParams fp;
    memset(&fp, 0, sizeof(fp));
    fp.M = M; fp.N = K; fp.out = (__nv_bfloat16*)dx;
    rc = M <= kNarrowRows ? launch_few_rows<kInput, false>(wt, 2L * F, dpre, 2 * F, fp, stream)
                          : launch_few_rows<kInput, true>(wt, 2L * F, dpre, 2 * F, fp, stream);
    if (rc != FP4AR_OK) return rc;
  } else if (dx) {
    Maps maps;
    memset(&maps, 0, sizeof(maps));
    memset(&p, 0, sizeof(p));
    if (!map_2d(&maps.a, dpre, M, 2L * F, 128) || !map_2d(&maps.b, wt, 2L * F, K, 64) || !map_2d(&maps.out, dx, M, K, 32)) return FP4AR_ERR_UNSUPPORTED;
    p.M = M; p.N = K; p.kblocks = (2 * F + 63) / 64;
    rc = launch_pair_gemm<kInput>(maps, p, stream);
    if (rc != FP4AR_OK) return rc;
  }
  if (dwt) {
    Maps maps;
    memset(&maps, 0, sizeof(maps));
    memset(&p, 0, sizeof(p));
    if (!map_2d(&maps.a, dpre, M, 2L * F, 64) || !map_2d(&maps.b, x, M, K, 64) || !map_2d(&maps.out, dwt, 2L * F, K, 32)) return FP4AR_ERR_UNSUPPORTED;
    p.M = 2 * F; p.N = K; p.kblocks = (M + 63) / 64;
    rc = launch_pair_gemm<kWeight>(maps, p, stream);
  }
  return rc;
}

extern "C" int fp4ar_layer_plan(int tiles, int kblocks, int units, int unit, int* used, int* segments, int max_segments) {
  if (tiles < 1 || kblocks < 1 || units < 1 || !used) return -1;
  const int cut = cut_units(tiles, kblocks, units), whole = tiles < units ? tiles : units;
  *used = cut > whole ? cut : whole;
  if (!segments) return 0;
  if (unit < 0 || unit >= *used) return -1;
  Walk walk(tiles, kblocks, unit, *used, cut);
  Seg s;
  int n = 0;
  for (; walk.next(s); n++)
    if (n < max_segments) {
      int* o = segments + 5 * n;
      o[0] = s.tile; o[1] = s.lo; o[2] = s.count; o[3] = s.kind; o[4] = s.others;
    }
  return n;
}
