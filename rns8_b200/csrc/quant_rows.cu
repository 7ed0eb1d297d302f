// Row quantisation to int8 (include/rns8/rns8_quant.h): one block a row, one
// pass over the row held in registers; rows too long for that are read twice.
// Bound by HBM: 8192 x 8192 bf16 32 us (6.3 TB/s), 4096 x 4096 f32 12.4 us (6.8);
// few rows by latency, 64 x 8192 bf16 1.7 us. The blocks past the rows align
// another matrix's rows, so that a product with unaligned weights starts after
// one launch, not two.
#include <algorithm>

#include "quant_common.cuh"
#include "quant_kernels.hpp"
#include "quant_launch.cuh"

namespace rns8cuda {
namespace {

// How a row is read: as 16-byte words; as the words around vectors of a row that
// starts anywhere, shifted into place; element by element.
enum class Read { Aligned, Shifted, Elements };

template <typename T, Read READ, int NV>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const T* __restrict__ x, int cols, int64_t ld_x,
                                                             int8_t* __restrict__ q, int64_t ld_q,
                                                             float* __restrict__ scale, int64_t rows,
                                                             const AlignRows align) {
  __shared__ uint32_t slots[32];
  wait_previous_launch();
  allow_next_launch();
  const int64_t row = blockIdx.x;
  if (row >= rows) {
    align_rows(align, (row - rows) * blockDim.x + threadIdx.x, (gridDim.x - rows) * blockDim.x);
    return;
  }
  const T* xr = x + row * ld_x;
  F2 v[NV][4];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (READ == Read::Shifted) {
      const Raw8<T> raw = load_shifted<T>(xr, cols, (j * blockDim.x + threadIdx.x) * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = raw.pair(e);
    } else {
      load8<READ == Read::Aligned>(xr, cols, j, blockDim.x, threadIdx.x, v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) top = max(top, magnitude_bits(v[j]));
  const RowScale rs = make_row_scale(block_max(top, slots));
  if (threadIdx.x == 0) scale[row] = rs.scale;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = (j * blockDim.x + threadIdx.x) * 8;
    if (READ != Read::Shifted || i + 8 <= cols) {
      store_q8<READ != Read::Elements>(q + row * ld_q, cols, j, blockDim.x, threadIdx.x, v[j], rs.inv);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < cols)
          q[row * ld_q + i + e] = static_cast<int8_t>(quantize_one(e % 2 ? v[j][e / 2].v.y : v[j][e / 2].v.x, rs.inv));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) quantize_long_rows_kernel(const T* __restrict__ x, int64_t cols, int64_t ld_x,
                                                                  int8_t* __restrict__ q, int64_t ld_q,
                                                                  float* __restrict__ scale, int64_t rows,
                                                                  const AlignRows align) {
  __shared__ uint32_t slots[32];
  wait_previous_launch();
  allow_next_launch();
  const int64_t row = blockIdx.x;
  if (row >= rows) {
    align_rows(align, (row - rows) * blockDim.x + threadIdx.x, (gridDim.x - rows) * blockDim.x);
    return;
  }
  const T* xr = x + row * ld_x;
  uint32_t top = 0;
  for (int64_t i = threadIdx.x; i < cols; i += blockDim.x) top = max(top, magnitude_bits(to_f32(xr[i])));
  const RowScale rs = make_row_scale(block_max(top, slots));
  if (threadIdx.x == 0) scale[row] = rs.scale;
  for (int64_t i = threadIdx.x; i < cols; i += blockDim.x)
    q[row * ld_q + i] = static_cast<int8_t>(quantize_one(to_f32(xr[i]), rs.inv));
}

template <typename T>
cudaError_t launch(const T* x, int64_t rows, int64_t cols, int64_t ld_x, int8_t* q, int64_t ld_q, float* scale,
                   const AlignRows* align, cudaStream_t stream) {
  const bool q_words = reinterpret_cast<uintptr_t>(q) % 8 == 0 && ld_q % 8 == 0;
  const bool aligned = q_words && cols % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_x * sizeof(T) % 16 == 0;
  // Blocks for the other matrix: 16 bytes a thread, four rounds of the GPU at most.
  auto grid = [&](unsigned threads) {
    int64_t blocks = 0;
    if (align) blocks = std::min<int64_t>((align->rows * (align->ld_dst / 16) + threads - 1) / threads, 4096);
    return dim3(static_cast<unsigned>(rows + blocks));
  };
  const AlignRows job = align ? *align : AlignRows{};
  if (cols > 1024 * 8 * 4)
    return launch_chained(quantize_long_rows_kernel<T>, grid(1024), 1024, 0, 1, stream, x, cols, ld_x, q, ld_q, scale,
                          rows, job);
  const int c = static_cast<int>(cols), vecs = (c + 7) / 8;
  auto go = [&](auto nv, auto read) {
    constexpr int NV = decltype(nv)::value;
    const unsigned threads = static_cast<unsigned>(std::max(32, ((vecs + NV - 1) / NV + 31) / 32 * 32));
    return launch_chained(quantize_rows_kernel<T, decltype(read)::value, NV>, grid(threads), threads, 0, 1, stream, x, c,
                          ld_x, q, ld_q, scale, rows, job);
  };
  auto pick = [&](auto read) {
    const int nv = row_vectors(rows, vecs);
    if (nv == 1) return go(std::integral_constant<int, 1>{}, read);
    if (nv == 2) return go(std::integral_constant<int, 2>{}, read);
    return go(std::integral_constant<int, 4>{}, read);
  };
  if (aligned) return pick(std::integral_constant<Read, Read::Aligned>{});
  // 1500 x 5713: bf16 8.0 us, f32 11.0; element by element 28 and 20.5.
  if (q_words) return pick(std::integral_constant<Read, Read::Shifted>{});
  return pick(std::integral_constant<Read, Read::Elements>{});
}

}  // namespace

cudaError_t quantize_rows(const void* x, uint32_t x_type, int64_t rows, int64_t cols, int64_t ld_x, int8_t* q,
                          int64_t ld_q, float* scale, cudaStream_t stream, const AlignRows* align) {
  switch (x_type) {
    case RNS8_CUDA_TYPE_BF16:
      return launch(static_cast<const __nv_bfloat16*>(x), rows, cols, ld_x, q, ld_q, scale, align, stream);
    case RNS8_CUDA_TYPE_F16:
      return launch(static_cast<const __half*>(x), rows, cols, ld_x, q, ld_q, scale, align, stream);
    default:
      return launch(static_cast<const float*>(x), rows, cols, ld_x, q, ld_q, scale, align, stream);
  }
}

}  // namespace rns8cuda
