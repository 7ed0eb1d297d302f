// Scaled int8 product for a few tokens, on the CUDA cores: a stream over the
// weights at HBM speed.
//
// A block owns a run of output channels. It first holds the tokens as int8 in
// shared memory (quantising floating rows itself, so one launch serves the
// whole layer), then its warps take units of 2048 weight bytes (ROWS rows x
// 2048 / ROWS bytes), four 16-byte loads a lane, fold them with dp4a against
// every token and add the warp's exact integer sums into the block's
// accumulators. A unit's loads are issued before the previous unit is folded,
// the first one's before the tokens are quantised.
#include <algorithm>
#include <atomic>

#include "device_common.cuh"
#include "linear_internal.hpp"
#include "quant_common.cuh"

namespace rns8cuda {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int TILE_ROWS = 256;  // output channels whose sums a block holds at once
constexpr int UNIT_LOADS = 4;   // 16-byte loads a lane has in flight for one unit

template <int TOKENS>
struct Shape {
  static constexpr int ROWS = TOKENS <= 2 ? 1 : (TOKENS <= 4 ? 2 : 4);  // weight rows that share a token word
  static constexpr int CHUNKS = UNIT_LOADS / ROWS;                      // 512-byte spans of each row
};

int64_t padded_k(int64_t k) { return (k + 15) / 16 * 16; }
int tokens_of(int64_t m) { return m <= 1 ? 1 : (m <= 2 ? 2 : (m <= 4 ? 4 : 8)); }

__device__ __forceinline__ uint4 load_weights(const int8_t* row, int64_t at, int64_t k) {
  if (at + 16 <= k) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(row + at));
    return v;
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int b = 0; b < 16; ++b)
    if (at + b < k) w[b / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(row[at + b])) << (8 * (b % 4));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// q[token][kp] in shared memory from floating rows; scales to s[token].
template <typename T, int TOKENS>
__device__ void quantize_tokens(const LinearArgs& p, int8_t* q, int kp, float* s, uint32_t* slots) {
  const int k = static_cast<int>(p.k), m = static_cast<int>(p.m);
  const T* x = static_cast<const T*>(p.a);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && p.ld_a * sizeof(T) % 16 == 0;
  constexpr int PER = 16 / sizeof(T);  // elements of a 16-byte load
  uint32_t top[TOKENS] = {};
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    if (t >= m) break;
    const T* row = x + t * p.ld_a;
    int i = threadIdx.x * PER;
    if (vec)
      for (; i + PER <= k; i += THREADS * PER) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + i);
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int j = 0; j < PER; ++j) top[t] = max(top[t], magnitude_bits(to_f32(e[j])));
      }
    for (; i < k; i += THREADS * PER)
      for (int j = 0; j < PER && i + j < k; ++j) top[t] = max(top[t], magnitude_bits(to_f32(row[i + j])));
  }
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    top[t] = __reduce_max_sync(0xFFFFFFFFu, top[t]);
    if (lane == 0) slots[t * WARPS + warp] = top[t];
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    const RowScale rs = make_row_scale(__reduce_max_sync(0xFFFFFFFFu, slots[t * WARPS + lane % WARPS]));
    if (threadIdx.x == 0) s[t] = rs.scale;
    const T* row = x + t * p.ld_a;
    // Four elements to a word; bytes past k, and tokens past m, are zero.
    for (int i = threadIdx.x * 4; i < kp; i += THREADS * 4) {
      uint32_t w = 0;
      if (t < m) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (vec && i + 4 <= k) {
          if (sizeof(T) == 4) {
            const float4 raw = *reinterpret_cast<const float4*>(row + i);
            v[0] = raw.x, v[1] = raw.y, v[2] = raw.z, v[3] = raw.w;
          } else {
            const uint2 raw = *reinterpret_cast<const uint2*>(row + i);
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = to_f32(e[j]);
          }
        } else {
          for (int j = 0; j < 4; ++j)
            if (i + j < k) v[j] = to_f32(row[i + j]);
        }
        // A non-finite row has inv = 0: past-the-end zeros stay zero.
#pragma unroll
        for (int j = 0; j < 4; ++j) w |= (static_cast<uint32_t>(quantize_one(v[j], rs.inv)) & 0xFFu) << (8 * j);
      }
      *reinterpret_cast<uint32_t*>(q + t * kp + i) = w;
    }
  }
}

template <int TOKENS>
__device__ void copy_tokens(const LinearArgs& p, int8_t* q, int kp, float* s) {
  const int k = static_cast<int>(p.k), m = static_cast<int>(p.m);
  const int8_t* a = static_cast<const int8_t*>(p.a);
  const bool words = reinterpret_cast<uintptr_t>(a) % 4 == 0 && p.ld_a % 4 == 0;
  for (int t = 0; t < TOKENS; ++t)
    for (int i = threadIdx.x * 4; i < kp; i += THREADS * 4) {
      uint32_t w = 0;
      if (t < m) {
        const int8_t* row = a + t * p.ld_a;
        if (words && i + 4 <= k)
          w = *reinterpret_cast<const uint32_t*>(row + i);
        else
          for (int j = 0; j < 4; ++j)
            if (i + j < k) w |= static_cast<uint32_t>(static_cast<uint8_t>(row[i + j])) << (8 * j);
      }
      *reinterpret_cast<uint32_t*>(q + t * kp + i) = w;
    }
  if (threadIdx.x < m) s[threadIdx.x] = p.a_scale[threadIdx.x];
}

__device__ __forceinline__ void store_any(void* out, uint32_t type, int64_t i, float v) {
  if (type == RNS8_CUDA_TYPE_BF16)
    static_cast<__nv_bfloat16*>(out)[i] = from_f32<__nv_bfloat16>(v);
  else if (type == RNS8_CUDA_TYPE_F16)
    static_cast<__half*>(out)[i] = from_f32<__half>(v);
  else
    static_cast<float*>(out)[i] = v;
}

template <int TOKENS, bool GATED>
__global__ void __launch_bounds__(THREADS) linear_gemv_kernel(const LinearArgs p, int kp) {
  using S = Shape<TOKENS>;
  constexpr int HALVES = GATED ? 2 : 1;
  extern __shared__ __align__(16) int8_t smem[];
  int8_t* q = smem;
  int* acc = reinterpret_cast<int*>(smem + TOKENS * kp);  // [HALVES][TILE_ROWS][TOKENS]
  __shared__ float s[TOKENS];
  __shared__ uint32_t slots[TOKENS * WARPS];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t first = p.n * blockIdx.x / gridDim.x, last = p.n * (blockIdx.x + 1) / gridDim.x;
  const int spans = (kp + 512 * S::CHUNKS - 1) / (512 * S::CHUNKS);  // units along k

  for (int64_t j0 = first; j0 < last; j0 += TILE_ROWS) {
    const int rows = static_cast<int>(min(last - j0, static_cast<int64_t>(TILE_ROWS)));
    const int groups = (rows + S::ROWS - 1) / S::ROWS;
    const int units = HALVES * groups * spans;
    uint4 next[S::ROWS][S::CHUNKS];
    auto fetch = [&](int u) {
      const int span = u % spans, hg = u / spans, half = hg / groups, r0 = (hg % groups) * S::ROWS;
#pragma unroll
      for (int r = 0; r < S::ROWS; ++r) {
        const int64_t row = min(j0 + r0 + r, last - 1) + half * p.n;  // a repeated row's sums are dropped
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
          const int64_t at = (static_cast<int64_t>(span) * S::CHUNKS + c) * 512 + lane * 16;
          next[r][c] = at < p.k ? load_weights(p.w + row * p.ld_w, at, p.k) : make_uint4(0, 0, 0, 0);
        }
      }
    };
    if (warp < units) fetch(warp);
    for (int i = threadIdx.x; i < HALVES * TILE_ROWS * TOKENS; i += THREADS) acc[i] = 0;
    if (j0 == first) {
      if (p.a_type == RNS8_CUDA_TYPE_I8)
        copy_tokens<TOKENS>(p, q, kp, s);
      else if (p.a_type == RNS8_CUDA_TYPE_BF16)
        quantize_tokens<__nv_bfloat16, TOKENS>(p, q, kp, s, slots);
      else if (p.a_type == RNS8_CUDA_TYPE_F16)
        quantize_tokens<__half, TOKENS>(p, q, kp, s, slots);
      else
        quantize_tokens<float, TOKENS>(p, q, kp, s, slots);
    }
    __syncthreads();
    for (int u = warp; u < units; u += WARPS) {
      uint4 w[S::ROWS][S::CHUNKS];
#pragma unroll
      for (int r = 0; r < S::ROWS; ++r)
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) w[r][c] = next[r][c];
      if (u + WARPS < units) fetch(u + WARPS);
      int sum[S::ROWS][TOKENS] = {};
      const int span = u % spans, hg = u / spans, half = hg / groups, r0 = (hg % groups) * S::ROWS;
#pragma unroll
      for (int c = 0; c < S::CHUNKS; ++c) {
        const int at = (span * S::CHUNKS + c) * 512 + lane * 16;
        if (at < kp) {
#pragma unroll
          for (int t = 0; t < TOKENS; ++t) {
            const uint4 x = *reinterpret_cast<const uint4*>(q + t * kp + at);
#pragma unroll
            for (int r = 0; r < S::ROWS; ++r) {
              sum[r][t] = __dp4a(static_cast<int>(w[r][c].x), static_cast<int>(x.x), sum[r][t]);
              sum[r][t] = __dp4a(static_cast<int>(w[r][c].y), static_cast<int>(x.y), sum[r][t]);
              sum[r][t] = __dp4a(static_cast<int>(w[r][c].z), static_cast<int>(x.z), sum[r][t]);
              sum[r][t] = __dp4a(static_cast<int>(w[r][c].w), static_cast<int>(x.w), sum[r][t]);
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < S::ROWS; ++r)
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
          const int total = __reduce_add_sync(0xFFFFFFFFu, sum[r][t]);
          if (lane == 0 && r0 + r < rows) atomicAdd(&acc[(half * TILE_ROWS + r0 + r) * TOKENS + t], total);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * TOKENS; i += THREADS) {
      const int t = i / rows, r = i % rows;
      if (t >= p.m) break;
      const int64_t j = j0 + r;
      float y = static_cast<float>(acc[r * TOKENS + t]) * s[t] * p.w_scale[j];
      if (p.bias) y += p.bias[j];
      if (GATED) {
        float up = static_cast<float>(acc[(TILE_ROWS + r) * TOKENS + t]) * s[t] * p.w_scale[p.n + j];
        if (p.bias) up += p.bias[p.n + j];
        y = y / (1.0f + expf(-y)) * up;
      }
      store_any(p.out, p.out_type, t * p.ld_out + j, y);
    }
    __syncthreads();
  }
}

template <int TOKENS, bool GATED>
size_t smem_bytes(int64_t k) {
  return static_cast<size_t>(TOKENS * padded_k(k) + (GATED ? 2 : 1) * TILE_ROWS * TOKENS * sizeof(int));
}

template <int TOKENS, bool GATED>
cudaError_t launch(const LinearArgs& p, int sm_count, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  const cudaError_t e = raise_smem_limit_once(linear_gemv_kernel<TOKENS, GATED>, 200 * 1024, configured);
  if (e != cudaSuccess) return e;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(p.n, sm_count));
  linear_gemv_kernel<TOKENS, GATED>
      <<<grid, THREADS, smem_bytes<TOKENS, GATED>(p.k), stream>>>(p, static_cast<int>(padded_k(p.k)));
  return cudaGetLastError();
}

}  // namespace

bool gemv_supported(const LinearArgs& p) {
  return p.m <= kGemvMaxTokens && reinterpret_cast<uintptr_t>(p.w) % 16 == 0 && p.ld_w % 16 == 0 &&
         tokens_of(p.m) * padded_k(p.k) <= 160 * 1024;
}

cudaError_t linear_gemv(const LinearArgs& p, int sm_count, cudaStream_t stream) {
  auto go = [&](auto gated) {
    constexpr bool G = decltype(gated)::value;
    switch (tokens_of(p.m)) {
      case 1: return launch<1, G>(p, sm_count, stream);
      case 2: return launch<2, G>(p, sm_count, stream);
      case 4: return launch<4, G>(p, sm_count, stream);
      default: return launch<8, G>(p, sm_count, stream);
    }
  };
  return p.gated ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace rns8cuda
