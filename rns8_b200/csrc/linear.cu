// Scaled int8 product (include/rns8/rns8_quant.h), first form: 64 x 64 output
// tiles on the CUDA cores with byte-wise operand loads, right for any
// alignment.
#include "quant_common.cuh"
#include "quant_kernels.hpp"

namespace rns8cuda {
namespace {

constexpr int TILE = 64, KT = 64;

__device__ __forceinline__ void store_out(void* out, uint32_t type, int64_t i, float v) {
  if (type == RNS8_CUDA_TYPE_BF16)
    static_cast<__nv_bfloat16*>(out)[i] = from_f32<__nv_bfloat16>(v);
  else if (type == RNS8_CUDA_TYPE_F16)
    static_cast<__half*>(out)[i] = from_f32<__half>(v);
  else
    static_cast<float*>(out)[i] = v;
}

struct LinearArgs {
  const int8_t* a;
  const int8_t* w;
  const float *a_scale, *w_scale, *bias;
  void* out;
  int64_t m, n, k, ld_a, ld_w, ld_out;
  uint32_t out_type, gated;
};

// 256 threads, 4 x 4 outputs each; a gated tile accumulates both halves.
__global__ void __launch_bounds__(256) linear_simt_kernel(LinearArgs p) {
  __shared__ int8_t as[TILE][KT + 4], ws[2][TILE][KT + 4];
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * TILE, n0 = static_cast<int64_t>(blockIdx.x) * TILE;
  const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
  const int halves = p.gated ? 2 : 1;
  int acc[2][4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += KT) {
    for (int i = threadIdx.x; i < TILE * KT; i += 256) {
      const int r = i / KT, c = i % KT;
      as[r][c] = (m0 + r < p.m && k0 + c < p.k) ? p.a[(m0 + r) * p.ld_a + k0 + c] : 0;
      for (int h = 0; h < halves; ++h)
        ws[h][r][c] = (n0 + r < p.n && k0 + c < p.k) ? p.w[(h * p.n + n0 + r) * p.ld_w + k0 + c] : 0;
    }
    __syncthreads();
    for (int c = 0; c < KT; c += 4)
      for (int h = 0; h < halves; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[h][i][j] = __dp4a(*reinterpret_cast<const int*>(&as[tr + 16 * i][c]),
                                  *reinterpret_cast<const int*>(&ws[h][tc + 16 * j][c]), acc[h][i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + tr + 16 * i, c = n0 + tc + 16 * j;
      if (r >= p.m || c >= p.n) continue;
      float y[2];
      for (int h = 0; h < halves; ++h) {
        const int64_t wr = h * p.n + c;
        y[h] = static_cast<float>(acc[h][i][j]) * p.a_scale[r] * p.w_scale[wr];
        if (p.bias) y[h] += p.bias[wr];
      }
      store_out(p.out, p.out_type, r * p.ld_out + c, p.gated ? y[0] / (1.0f + expf(-y[0])) * y[1] : y[0]);
    }
}

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

}  // namespace

uint64_t linear_scratch_bytes(const rns8_cuda_linear_desc& d, int) {
  if (d.a_type == RNS8_CUDA_TYPE_I8) return 0;
  return round_up(static_cast<uint64_t>(d.m) * round_up(d.k, 16), 256) + round_up(4ull * d.m, 256);
}

cudaError_t linear(const rns8_cuda_linear_desc& d, int, cudaStream_t stream) {
  LinearArgs p{static_cast<const int8_t*>(d.a), d.w, d.a_scale, d.w_scale, d.bias, d.out, d.m, d.n, d.k, d.ld_a, d.ld_w,
               d.ld_out, d.out_type, d.flags & RNS8_CUDA_LINEAR_GATED};
  if (d.a_type != RNS8_CUDA_TYPE_I8) {
    const int64_t ld = static_cast<int64_t>(round_up(d.k, 16));
    int8_t* q = static_cast<int8_t*>(d.scratch);
    float* s = reinterpret_cast<float*>(q + round_up(static_cast<uint64_t>(d.m) * ld, 256));
    const cudaError_t e = quantize_rows(d.a, d.a_type, d.m, d.k, d.ld_a, q, ld, s, stream);
    if (e != cudaSuccess) return e;
    p.a = q;
    p.ld_a = ld;
    p.a_scale = s;
  }
  const dim3 grid(static_cast<unsigned>((d.n + TILE - 1) / TILE), static_cast<unsigned>((d.m + TILE - 1) / TILE));
  linear_simt_kernel<<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace rns8cuda
