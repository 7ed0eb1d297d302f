// Internal launch API of the 8-bit operators (include/rns8/rns8_quant.h).
// Arguments are validated by the callers in api_quant.cpp; every function
// enqueues on `stream` and returns the launch's error.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "rns8/rns8_quant.h"

namespace rns8cuda {

// The limit of the kernels' waits (rns8_cuda_quant_wait_limit), usual and now.
constexpr int64_t kQuantWaitCycles = 4000000000;
int64_t quant_wait_cycles();

// With `align` the same launch also copies another int8 matrix's rows to
// 16-byte boundaries (quant_common.cuh).
struct AlignRows;
cudaError_t quantize_rows(const void* x, uint32_t x_type, int64_t rows, int64_t cols, int64_t ld_x, int8_t* q,
                          int64_t ld_q, float* scale, cudaStream_t stream, const AlignRows* align = nullptr);

uint64_t linear_scratch_bytes(const rns8_cuda_linear_desc& d);
// Tokens to a tile and blocks to a cluster; tile 0: tokens on lanes.
struct LinearForm {
  uint32_t tile, splits;
};
LinearForm linear_form(const rns8_cuda_linear_desc& d, int sm_count);
cudaError_t linear(const rns8_cuda_linear_desc& d, int sm_count, cudaStream_t stream);

cudaError_t residual_norm(const rns8_cuda_residual_norm_desc& d, int sm_count, cudaStream_t stream);
uint64_t residual_norm_backward_scratch_bytes(const rns8_cuda_residual_norm_backward_desc& d, int sm_count);
cudaError_t residual_norm_backward(const rns8_cuda_residual_norm_backward_desc& d, int sm_count, cudaStream_t stream);

}  // namespace rns8cuda
