// C entry points of the 8-bit operators (include/rns8/rns8_quant.h): argument
// checks, then the launch on the caller's device and stream.
#include <atomic>

#include "api_internal.hpp"
#include "quant_kernels.hpp"

namespace {

// Sizes stay below 2^31 rows or columns and every matrix below 2^60 bytes, so
// no offset computed from them overflows 64 bits.
constexpr int64_t kMaxExtent = (int64_t{1} << 31) - 1;
constexpr int64_t kMaxElements = int64_t{1} << 57;

template <typename D>
bool valid_header(const D* d) {
  return d && d->struct_size >= sizeof(D) && d->abi_version == RNS8_ABI_VERSION;
}

bool float_type(uint32_t t) { return t <= RNS8_CUDA_TYPE_F32; }
uint32_t type_size(uint32_t t) { return t == RNS8_CUDA_TYPE_F32 ? 4 : (t == RNS8_CUDA_TYPE_I8 ? 1 : 2); }
bool aligned_to(const void* p, uint32_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

bool valid_rows(const void* p, int64_t rows, int64_t cols, int64_t ld, uint32_t elem) {
  return p && aligned_to(p, elem) && ld >= cols && ld <= kMaxElements / (rows > 0 ? rows : 1);
}

// Multiprocessors of a device, asked once per device.
int sm_count_of(int device_id) {
  static std::atomic<int> known[64];
  const bool slot = device_id >= 0 && device_id < 64;
  int count = slot ? known[device_id].load(std::memory_order_relaxed) : 0;
  if (count > 0) return count;
  if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device_id) != cudaSuccess || count <= 0) {
    (void)cudaGetLastError();
    return 148;
  }
  if (slot) known[device_id].store(count, std::memory_order_relaxed);
  return count;
}

rns8_status launch_result(cudaError_t e) {
  if (e == cudaErrorInvalidValue) return RNS8_INVALID_ARGUMENT;
  return rns8host::cuda_status(e);
}

rns8_status check_linear(const rns8_cuda_linear_desc* d) {
  if (!valid_header(d) || (d->flags & ~RNS8_CUDA_LINEAR_GATED) || d->reserved) return RNS8_INVALID_ARGUMENT;
  if (d->a_type > RNS8_CUDA_TYPE_I8 || d->out_type > RNS8_CUDA_TYPE_I8) return RNS8_INVALID_ARGUMENT;
  if (d->m < 0 || d->n < 1 || d->k < 1 || d->m > kMaxExtent || d->n > kMaxExtent / 2 || d->k > kMaxExtent)
    return RNS8_INVALID_ARGUMENT;
  const int64_t w_rows = (d->flags & RNS8_CUDA_LINEAR_GATED) ? 2 * d->n : d->n;
  if (!valid_rows(d->w, w_rows, d->k, d->ld_w, 1) || !d->w_scale || !aligned_to(d->w_scale, 4) ||
      !aligned_to(d->bias, 4))
    return RNS8_INVALID_ARGUMENT;
  if ((d->a_type == RNS8_CUDA_TYPE_I8) != (d->a_scale != nullptr) || !aligned_to(d->a_scale, 4))
    if (d->m > 0 || d->a_type != RNS8_CUDA_TYPE_I8) return RNS8_INVALID_ARGUMENT;
  if (d->m > 0 && (!valid_rows(d->a, d->m, d->k, d->ld_a, type_size(d->a_type)) ||
                   !valid_rows(d->out, d->m, d->n, d->ld_out, type_size(d->out_type))))
    return RNS8_INVALID_ARGUMENT;
  if (!aligned_to(d->out_scale, 4) || (d->m > 0 && (d->out_type == RNS8_CUDA_TYPE_I8) != (d->out_scale != nullptr)))
    return RNS8_INVALID_ARGUMENT;
  return d->k > RNS8_CUDA_LINEAR_MAX_K ? RNS8_ACCUMULATION_OVERFLOW_RISK : RNS8_SUCCESS;
}

// Types, sizes and parameters shared by the forward and backward descriptors.
template <typename D>
bool valid_norm(const D& d, uint32_t flags) {
  if ((d.flags & ~flags) || !float_type(d.type) || (d.weight_type != d.type && d.weight_type != RNS8_CUDA_TYPE_F32)) return false;
  if (d.tokens < 0 || d.tokens > kMaxExtent || d.dim < 1 || d.dim > 32768) return false;
  if (!(d.eps >= 0.0f) || d.eps > 3.4e38f) return false;
  const uint32_t w = type_size(d.weight_type);
  if (!aligned_to(d.post_weight, w) || !aligned_to(d.pre_weight, w)) return false;
  if (d.gate && d.tokens > 0 &&
      (d.groups < 1 || d.tokens % d.groups != 0 || !valid_rows(d.gate, d.groups, d.dim, d.ld_gate, w)))
    return false;
  return true;
}

bool valid_backward(const rns8_cuda_residual_norm_backward_desc& d) {
  if (!valid_norm(d, RNS8_CUDA_NORM_D_GATE_F32) || !aligned_to(d.d_post, 4) || !aligned_to(d.d_pre, 4)) return false;
  const bool gate_f32 = d.flags & RNS8_CUDA_NORM_D_GATE_F32;
  if (gate_f32 && d.weight_type != RNS8_CUDA_TYPE_F32) return false;
  if ((d.d_post && !d.post_weight) || (d.d_pre && !d.pre_weight) || (d.d_gate && !d.gate)) return false;
  if (d.tokens == 0) return !d.d_gate || (d.groups >= 0 && valid_rows(d.d_gate, d.groups, d.dim, d.ld_d_gate, 4));
  const uint32_t e = type_size(d.type);
  auto optional_rows = [&](const void* p, int64_t ld) { return !p || valid_rows(p, d.tokens, d.dim, ld, e); };
  if (!optional_rows(d.d_x_out, d.ld_d_x_out) || !optional_rows(d.d_h, d.ld_d_h)) return false;
  if (!valid_rows(d.x_out, d.tokens, d.dim, d.ld_x_out, e) || !valid_rows(d.y, d.tokens, d.dim, d.ld_y, e) ||
      !valid_rows(d.d_x, d.tokens, d.dim, d.ld_d_x, e) || !valid_rows(d.d_y, d.tokens, d.dim, d.ld_d_y, e))
    return false;
  return !d.d_gate || valid_rows(d.d_gate, d.groups, d.dim, d.ld_d_gate, d.groups == d.tokens && !gate_f32 ? e : 4);
}

}  // namespace

namespace {
std::atomic<int64_t> wait_cycles{rns8cuda::kQuantWaitCycles};
}  // namespace
int64_t rns8cuda::quant_wait_cycles() { return wait_cycles.load(std::memory_order_relaxed); }

extern "C" rns8_status rns8_cuda_quant_wait_limit(uint64_t cycles) {
  if (cycles > static_cast<uint64_t>(rns8cuda::kQuantWaitCycles)) return RNS8_INVALID_ARGUMENT;
  wait_cycles.store(cycles ? static_cast<int64_t>(cycles) : rns8cuda::kQuantWaitCycles, std::memory_order_relaxed);
  return RNS8_SUCCESS;
}

extern "C" rns8_status rns8_cuda_quantize_rows_device(const rns8_cuda_quantize_desc* desc) {
  if (!valid_header(desc) || desc->flags || !float_type(desc->x_type)) return RNS8_INVALID_ARGUMENT;
  const auto& d = *desc;
  if (d.rows < 0 || d.rows > kMaxExtent || d.cols < 1 || d.cols > kMaxExtent) return RNS8_INVALID_ARGUMENT;
  if (d.rows == 0) return RNS8_SUCCESS;
  if (!valid_rows(d.x, d.rows, d.cols, d.ld_x, type_size(d.x_type)) || !valid_rows(d.q, d.rows, d.cols, d.ld_q, 1) ||
      !d.scale || !aligned_to(d.scale, 4))
    return RNS8_INVALID_ARGUMENT;
  rns8host::DeviceScope scope(d.device_id);
  if (!scope.ok) return RNS8_BACKEND_FAILURE;
  return launch_result(rns8cuda::quantize_rows(d.x, d.x_type, d.rows, d.cols, d.ld_x, d.q, d.ld_q, d.scale,
                                               static_cast<cudaStream_t>(d.stream)));
}

extern "C" uint64_t rns8_cuda_linear_scratch_bytes(const rns8_cuda_linear_desc* desc) {
  if (check_linear(desc) != RNS8_SUCCESS || desc->m == 0) return 0;
  return rns8cuda::linear_scratch_bytes(*desc);
}

extern "C" rns8_status rns8_cuda_linear_device(const rns8_cuda_linear_desc* desc) {
  const rns8_status c = check_linear(desc);
  if (c != RNS8_SUCCESS) return c;
  if (!desc->status || !aligned_to(desc->status, 4)) return RNS8_INVALID_ARGUMENT;
  if (desc->m == 0) return RNS8_SUCCESS;
  rns8host::DeviceScope scope(desc->device_id);
  if (!scope.ok) return RNS8_BACKEND_FAILURE;
  const uint64_t need = rns8cuda::linear_scratch_bytes(*desc);
  if (need && (!desc->scratch || desc->scratch_bytes < need)) return RNS8_WORKSPACE_TOO_SMALL;
  return launch_result(rns8cuda::linear(*desc, sm_count_of(desc->device_id), static_cast<cudaStream_t>(desc->stream)));
}

extern "C" rns8_status rns8_cuda_linear_form(const rns8_cuda_linear_desc* desc, int32_t sm_count, uint32_t* tile,
                                             uint32_t* splits) {
  const rns8_status c = check_linear(desc);
  if (c != RNS8_SUCCESS) return c;
  if (sm_count < 1 || desc->m < 1 || !tile || !splits) return RNS8_INVALID_ARGUMENT;
  const rns8cuda::LinearForm f = rns8cuda::linear_form(*desc, sm_count);
  *tile = f.tile;
  *splits = f.splits;
  return RNS8_SUCCESS;
}

extern "C" rns8_status rns8_cuda_residual_norm_device(const rns8_cuda_residual_norm_desc* desc) {
  if (!valid_header(desc) || !valid_norm(*desc, 0)) return RNS8_INVALID_ARGUMENT;
  const auto& d = *desc;
  if (!d.pre_weight && (d.h || d.q)) return RNS8_INVALID_ARGUMENT;
  if (d.pre_weight && !d.h && !d.q && d.tokens > 0) return RNS8_INVALID_ARGUMENT;
  if (d.tokens == 0) return RNS8_SUCCESS;
  const uint32_t e = type_size(d.type);
  if (!valid_rows(d.x, d.tokens, d.dim, d.ld_x, e) || !valid_rows(d.y, d.tokens, d.dim, d.ld_y, e) ||
      !valid_rows(d.x_out, d.tokens, d.dim, d.ld_x_out, e) || (d.h && !valid_rows(d.h, d.tokens, d.dim, d.ld_h, e)) ||
      (d.q && (!valid_rows(d.q, d.tokens, d.dim, d.ld_q, 1) || !d.q_scale || !aligned_to(d.q_scale, 4))))
    return RNS8_INVALID_ARGUMENT;
  rns8host::DeviceScope scope(d.device_id);
  if (!scope.ok) return RNS8_BACKEND_FAILURE;
  return launch_result(rns8cuda::residual_norm(d, sm_count_of(d.device_id), static_cast<cudaStream_t>(d.stream)));
}

extern "C" uint64_t
rns8_cuda_residual_norm_backward_scratch_bytes(const rns8_cuda_residual_norm_backward_desc* desc) {
  if (!valid_header(desc) || !valid_backward(*desc) || desc->tokens == 0) return 0;
  return rns8cuda::residual_norm_backward_scratch_bytes(*desc, sm_count_of(desc->device_id));
}

extern "C" rns8_status
rns8_cuda_residual_norm_backward_device(const rns8_cuda_residual_norm_backward_desc* desc) {
  if (!valid_header(desc) || !valid_backward(*desc)) return RNS8_INVALID_ARGUMENT;
  const auto& d = *desc;
  const cudaStream_t stream = static_cast<cudaStream_t>(d.stream);
  rns8host::DeviceScope scope(d.device_id);
  if (!scope.ok) return RNS8_BACKEND_FAILURE;
  if (d.tokens == 0) {  // sums over no tokens
    for (float* g : {d.d_post, d.d_pre})
      if (g) {
        const cudaError_t e = cudaMemsetAsync(g, 0, static_cast<size_t>(d.dim) * sizeof(float), stream);
        if (e != cudaSuccess) return launch_result(e);
      }
    if (d.d_gate && d.groups > 0)
      return launch_result(cudaMemset2DAsync(d.d_gate, static_cast<size_t>(d.ld_d_gate) * sizeof(float), 0,
                                             static_cast<size_t>(d.dim) * sizeof(float),
                                             static_cast<size_t>(d.groups), stream));
    return RNS8_SUCCESS;
  }
  const int sms = sm_count_of(d.device_id);
  const uint64_t need = rns8cuda::residual_norm_backward_scratch_bytes(d, sms);
  if (need && (!d.scratch || d.scratch_bytes < need)) return RNS8_WORKSPACE_TOO_SMALL;
  return launch_result(rns8cuda::residual_norm_backward(d, sms, stream));
}
