// Shared by the kernels of the scaled int8 product (linear*.cu).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "rns8/rns8_quant.h"

namespace rns8cuda {

// One product: int8 rows of a with their scales, int8 rows of w.
struct LinearArgs {
  const int8_t* a;
  const int8_t* w;
  const float *a_scale, *w_scale, *bias;
  void* out;
  int64_t m, n, k, ld_a, ld_w, ld_out;
  uint32_t out_type;
  bool gated;
  bool after_quantize;  // the previous launch on the stream wrote a and a_scale, and nothing else that is read here
  uint32_t* status;
};

// The product (linear_tc.cu); rows of a and w 16-byte aligned.
cudaError_t linear_tc(const LinearArgs& p, int sm_count, cudaStream_t stream);

}  // namespace rns8cuda
