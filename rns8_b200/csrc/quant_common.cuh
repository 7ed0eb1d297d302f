// Shared by the 8-bit operators (row quantisation, scaled product, residual
// norms): element types, rows held in registers, block reductions and the
// quantisation rule.
//
// A row kernel gives every thread NV vectors of 8 elements. With ALIGNED rows
// (base and leading dimension on 16-byte boundaries) vector v of thread t
// covers elements 8 * (v * threads + t) .. + 7 and moves as 16-byte words;
// otherwise its e-th element is (8 v + e) * threads + t, so that a warp's
// element-wise accesses are contiguous. Elements past the row read as zero.
#pragma once

#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace rns8cuda {

// ---- element conversions -------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Vectors of 8 a thread of a row kernel holds. Few rows are a matter of latency:
// one vector a thread. With rows for every SM, blocks of at most 256 threads
// let the loads of one row run under the reductions of the others.
inline int row_vectors(int64_t rows, int vecs) {
  if (vecs > 1024) return 4;
  if (rows < 256 || vecs <= 256) return 1;
  return vecs <= 512 ? 2 : 4;
}

// Index of element (v, e) of this thread's part of a row.
template <bool ALIGNED>
__device__ __forceinline__ int row_index(int v, int e, int threads, int tid) {
  return ALIGNED ? (v * threads + tid) * 8 + e : (v * 8 + e) * threads + tid;
}

// Eight elements as 32-bit floats; elements at or past `cols` are zero.
template <bool ALIGNED, typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int cols, int v, int threads, int tid, float (&out)[8]) {
  if (ALIGNED) {
    const int i = (v * threads + tid) * 8;
    if (i + 8 <= cols) {
      constexpr int WORDS = static_cast<int>(sizeof(T) * 8 / 16);
      uint4 raw[WORDS];
#pragma unroll
      for (int w = 0; w < WORDS; ++w) raw[w] = reinterpret_cast<const uint4*>(row + i)[w];
      const T* t = reinterpret_cast<const T*>(raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = to_f32(t[e]);
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = row_index<ALIGNED>(v, e, threads, tid);
    out[e] = i < cols ? to_f32(row[i]) : 0.0f;
  }
}

template <bool ALIGNED, typename T>
__device__ __forceinline__ void store8(T* __restrict__ row, int cols, int v, int threads, int tid, const float (&in)[8]) {
  if (ALIGNED) {
    const int i = (v * threads + tid) * 8;
    if (i + 8 <= cols) {
      constexpr int WORDS = static_cast<int>(sizeof(T) * 8 / 16);
      uint4 raw[WORDS];
      T* t = reinterpret_cast<T*>(raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = from_f32<T>(in[e]);
#pragma unroll
      for (int w = 0; w < WORDS; ++w) reinterpret_cast<uint4*>(row + i)[w] = raw[w];
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = row_index<ALIGNED>(v, e, threads, tid);
    if (i < cols) row[i] = from_f32<T>(in[e]);
  }
}

// ---- quantisation rule ------------------------------------------------------------
// Magnitudes are compared by their bits: for non-negative floats the unsigned
// order of the bits is the numeric order, and a NaN is above everything, so a
// row's maximum is NaN when it holds one.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

struct RowScale {
  float scale, inv;
};
// scale = a / 127 and its inverse 127 / a. Below 127 * 2^-126 the scale would
// be subnormal and 127 / a could overflow: such rows count as zero rows. For a
// non-finite a the scale is a and every q is zero.
__device__ __forceinline__ RowScale make_row_scale(uint32_t max_bits) {
  const float a = __uint_as_float(max_bits);
  RowScale r;
  if (max_bits >= 0x7F800000u) {
    r.scale = a;
    r.inv = 0.0f;
  } else if (a < 127.0f * FLT_MIN) {
    r.scale = 0.0f;
    r.inv = 0.0f;
  } else {
    r.scale = __fdiv_rn(a, 127.0f);
    r.inv = __fdiv_rn(127.0f, a);
  }
  return r;
}
// |x * inv| <= 127 (1 + 2^-22), which rounds to at most 127. With inv = 0 the
// product of an infinity or a NaN is a NaN, which converts to 0.
__device__ __forceinline__ int quantize_one(float x, float inv) { return __float2int_rn(x * inv); }

template <bool ALIGNED>
__device__ __forceinline__ void store_q8(int8_t* __restrict__ row, int cols, int v, int threads, int tid,
                                         const float (&in)[8], float inv) {
  if (ALIGNED) {
    const int i = (v * threads + tid) * 8;
    if (i + 8 <= cols) {
      uint32_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t q0 = quantize_one(in[4 * h], inv), q1 = quantize_one(in[4 * h + 1], inv);
        const uint32_t q2 = quantize_one(in[4 * h + 2], inv), q3 = quantize_one(in[4 * h + 3], inv);
        w[h] = __byte_perm(__byte_perm(q0, q1, 0x0040), __byte_perm(q2, q3, 0x0040), 0x5410);
      }
      *reinterpret_cast<uint2*>(row + i) = make_uint2(w[0], w[1]);
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = row_index<ALIGNED>(v, e, threads, tid);
    if (i < cols) row[i] = static_cast<int8_t>(quantize_one(in[e], inv));
  }
}

// ---- block reductions ---------------------------------------------------------------
// One barrier each: every warp leaves its part in `slots` (32 words per value)
// and then sums all of them itself. Two reductions that follow one another use
// different slots.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* slots) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 16; o; o >>= 1) v[n] += __shfl_xor_sync(0xFFFFFFFFu, v[n], o);
  if (warps == 1) return;
  if (lane == 0)
#pragma unroll
    for (int n = 0; n < N; ++n) slots[n * 32 + warp] = v[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = lane < warps ? slots[n * 32 + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v[n] += __shfl_xor_sync(0xFFFFFFFFu, v[n], o);
  }
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* slots) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if (warps == 1) return v;
  if (lane == 0) slots[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xFFFFFFFFu, lane < warps ? slots[lane] : 0u);
}

}  // namespace rns8cuda
