// Scaled int8 product (include/rns8/rns8_quant.h): which kernels a call runs,
// the copies that give unaligned rows a 16-byte start, and the scratch for them.
#include <algorithm>

#include "linear_internal.hpp"
#include "quant_common.cuh"
#include "quant_kernels.hpp"
#include "quant_launch.cuh"

namespace rns8cuda {
namespace {

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }
bool aligned16(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 16 == 0; }

__global__ void __launch_bounds__(256) align_rows_kernel(const AlignRows job) {
  wait_previous_launch();
  allow_next_launch();
  align_rows(job, static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x,
             static_cast<int64_t>(gridDim.x) * blockDim.x);
}
cudaError_t launch_align(const AlignRows& job, int sm_count, cudaStream_t stream) {
  const int64_t chunks = job.rows * (job.ld_dst / 16);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((chunks + 255) / 256, sm_count * 16));
  return launch_chained(align_rows_kernel, dim3(grid), 256, 0, 1, stream, job);
}

// What a call needs around its product, and where in scratch.
struct Steps {
  bool align_w, align_a, quantize, quantize_out;
  int64_t w_rows, ld;
  uint64_t at_a, at_scale, at_out, bytes;
};
Steps plan(const rns8_cuda_linear_desc& d) {
  Steps s{};
  s.w_rows = (d.flags & RNS8_CUDA_LINEAR_GATED) ? 2 * d.n : d.n;
  s.ld = static_cast<int64_t>(round_up(d.k, 16));
  s.align_w = !aligned16(d.w, d.ld_w);
  s.quantize = d.a_type != RNS8_CUDA_TYPE_I8;
  s.align_a = !s.quantize && !aligned16(d.a, d.ld_a);
  if (s.align_w) s.bytes = round_up(static_cast<uint64_t>(s.w_rows) * s.ld, 256);
  s.at_a = s.bytes;
  if (s.quantize || s.align_a) s.bytes += round_up(static_cast<uint64_t>(d.m) * s.ld, 256);
  s.at_scale = s.bytes;
  if (s.quantize) s.bytes += round_up(4ull * d.m, 256);
  s.at_out = s.bytes;
  s.quantize_out = d.out_type == RNS8_CUDA_TYPE_I8;
  if (s.quantize_out) s.bytes += 4ull * static_cast<uint64_t>(d.m) * round_up(d.n, 4);
  if (s.bytes) s.bytes += 256;  // the caller's scratch may start anywhere
  return s;
}

}  // namespace

uint64_t linear_scratch_bytes(const rns8_cuda_linear_desc& d) { return plan(d).bytes; }

cudaError_t linear(const rns8_cuda_linear_desc& d, int sm_count, cudaStream_t stream) {
  const Steps s = plan(d);
  LinearArgs p{static_cast<const int8_t*>(d.a), d.w, d.a_scale, d.w_scale, d.bias, d.out, d.m, d.n, d.k, d.ld_a, d.ld_w,
               d.ld_out, d.out_type, (d.flags & RNS8_CUDA_LINEAR_GATED) != 0, false, d.status};
  int8_t* scratch = reinterpret_cast<int8_t*>(round_up(reinterpret_cast<uintptr_t>(d.scratch), 256));
  cudaError_t e = cudaSuccess;
  const AlignRows weights{d.w, scratch, s.w_rows, d.k, d.ld_w, s.ld};
  if (s.align_w) {
    p.w = scratch;
    p.ld_w = s.ld;
    if (!s.quantize) e = launch_align(weights, sm_count, stream);
  }
  if (e == cudaSuccess && (s.align_a || s.quantize)) {
    int8_t* q = scratch + s.at_a;
    float* scale = reinterpret_cast<float*>(scratch + s.at_scale);
    if (s.quantize) {
      e = quantize_rows(d.a, d.a_type, d.m, d.k, d.ld_a, q, s.ld, scale, stream, s.align_w ? &weights : nullptr);
      p.a_scale = scale;
      p.after_quantize = !s.align_w;
    } else {
      e = launch_align(AlignRows{p.a, q, d.m, d.k, d.ld_a, s.ld}, sm_count, stream);
    }
    p.a = q;
    p.ld_a = s.ld;
  }
  if (e != cudaSuccess) return e;
  if (!s.quantize_out) return linear_tc(p, sm_count, stream);
  p.out = scratch + s.at_out;
  p.out_type = RNS8_CUDA_TYPE_F32;
  p.ld_out = static_cast<int64_t>(round_up(d.n, 4));
  e = linear_tc(p, sm_count, stream);
  if (e != cudaSuccess) return e;
  return quantize_rows(p.out, RNS8_CUDA_TYPE_F32, d.m, d.n, p.ld_out, static_cast<int8_t*>(d.out), d.ld_out, d.out_scale,
                       stream);
}

}  // namespace rns8cuda
