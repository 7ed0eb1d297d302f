// Shared by the kernels of the scaled int8 product (linear*.cu).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "rns8/rns8_quant.h"

namespace rns8cuda {

// One product: int8 rows of a with their scales (or, where a kernel says so,
// floating rows of a_type that it quantises itself), int8 rows of w.
struct LinearArgs {
  const void* a;
  const int8_t* w;
  const float *a_scale, *w_scale, *bias;
  void* out;
  int64_t m, n, k, ld_a, ld_w, ld_out;
  uint32_t a_type, out_type;
  bool gated;
  bool after_quantize;  // the previous launch on the stream wrote a and a_scale
  uint32_t* status;
};

// Few tokens, CUDA cores (linear_gemv.cu).
constexpr int kGemvMaxTokens = 8;
bool gemv_supported(const LinearArgs& p);
cudaError_t linear_gemv(const LinearArgs& p, int sm_count, cudaStream_t stream);

// Tensor cores (linear_tc.cu); a int8, rows of a and w 16-byte aligned.
cudaError_t linear_tc(const LinearArgs& p, int sm_count, cudaStream_t stream);

}  // namespace rns8cuda
