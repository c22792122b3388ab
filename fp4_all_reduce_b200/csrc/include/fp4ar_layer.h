/* The feed-forward half of a tensor-parallel layer (B200, tcgen05 / TMEM): gated projections with their backward pass, and the
 * row-parallel linear with low-rank adapters of many requests.  BF16 in and out, FP32 sums.
 *
 * Everything is asynchronous on `stream`, takes its workspaces from the caller and can be captured.  Pointers are 16-byte
 * aligned, rows contiguous; M = 0 launches nothing (the weight gradient is then cleared).  The waits inside the GEMM kernels are
 * bounded and report to fp4ar_gemm_status().
 */
#ifndef FP4AR_LAYER_H_
#define FP4AR_LAYER_H_

#include "fp4ar.h"

#ifdef __cplusplus
extern "C" {
#endif

/* a(g): g sigmoid(g);  g Phi(g) (normal distribution);  its form with tanh */
enum { FP4AR_ACT_SILU = 0, FP4AR_ACT_GELU = 1, FP4AR_ACT_GELU_TANH = 2 };

/* h[M,F] = a(x Wg^T) * (x Wu^T), x [M,K], wt [2F,K]: the F gate rows, then the F up rows.  K and F are multiples of 8.
 * pre: optional [M,2F] FP32, the two projections (what the backward pass takes). */
int fp4ar_gated_linear(const void* x, const void* wt, int M, int F, int K, int act, void* h, void* pre, fp4ar_stream stream);

/* Gradients of h for dh [M,F].  dpre [M,2F] BF16 is written: (dh up a'(gate), dh a(gate)); then
 * dx [M,K] = dpre wt (or NULL) and dwt [2F,K] = dpre^T x (or NULL).  x is needed for dwt only, wt for dx only. */
int fp4ar_gated_backward(const void* dh, const void* pre, const void* x, const void* wt, int M, int F, int K, int act, void* dpre,
                         void* dx, void* dwt, fp4ar_stream stream);

/* y[M,N] = x Wt^T + scales[i] (x A_i^T) B_i^T, i = ids[row]; rows whose id is outside 0 .. adapters-1 have no adapter.
 * a [adapters,R,K], b [adapters,N,R], scales [adapters] FP32 or NULL (1.0).  K, N and R are multiples of 8, R <= 128.
 * A row depends on its own adapter only, whatever another request's adapter holds (infinities and NaN included).
 * workspace: fp4ar_adapters_workspace() bytes, not used by any other call until this one has run. */
size_t fp4ar_adapters_workspace(int M, int R, int adapters);
int fp4ar_linear_adapters(const void* x, const void* wt, const int* ids, const void* a, const void* b, const float* scales, int M, int N,
                          int K, int R, int adapters, void* workspace, void* y, fp4ar_stream stream);

/* Which kernel takes a call of fp4ar_linear_adapters (host only): 1 the one for few rows, 0 tiles of 256 rows, -1 for bad arguments. */
int fp4ar_adapters_few_rows(int M, int adapters);

/* How these products share their work (host only): `tiles` output tiles of `kblocks` K blocks over `units` CTA pairs.  *used: units that
 * work.  With `segments` the work of `unit` as (tile, first K block, K blocks, kind: 0 whole, 1 leaves a partial, 2 finishes the
 * tile, units that leave partials for it); returns the number of segments (also beyond max_segments), -1 for bad arguments. */
int fp4ar_layer_plan(int tiles, int kblocks, int units, int unit, int* used, int* segments, int max_segments);

#ifdef __cplusplus
}
#endif
#endif /* FP4AR_LAYER_H_ */
