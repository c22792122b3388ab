// The workspace of a GEMM launch whose K loops are cut over CTAs: one slot of 128 x 256 floats and kSplitFlags flags per SM, all flags zero
// between launches.  One per stream and one per captured graph (see StreamKSpace in gemm_fp4.cu); held until the launch is enqueued.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace fp4ar {

constexpr int kSplitFlags = 8;
class StreamKLease;
class SplitSpace {
 public:
  explicit SplitSpace(cudaStream_t stream);
  ~SplitSpace();
  SplitSpace(const SplitSpace&) = delete;
  SplitSpace& operator=(const SplitSpace&) = delete;
  float* partial() const;        // null: none could be had
  uint32_t* flags() const;

 private:
  StreamKLease* lease_;
};

}  // namespace fp4ar
