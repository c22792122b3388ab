// Host side of the tensor maps: the driver's encoder, looked up once, and the status block that every GEMM kernel reports to.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <mutex>

namespace fp4ar {

struct StatusWords;
StatusWords* gemm_status_word();      // of the current device, allocated by the first thread that needs it (null: out of memory)

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}
// Encodes a map.  The driver's function wants a context that is current to the calling thread, which a thread whose first CUDA call this
// is does not have yet; cudaSetDevice makes it so (during a capture too).
template <class... A>
bool encode_tiled(A... args) {
  const EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  if (fn(args...) == CUDA_SUCCESS) return true;
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess && fn(args...) == CUDA_SUCCESS;
}

}  // namespace fp4ar
