// The norms around a block fused with its gate and residual update, forward
// and backward (include/rns8/rns8_quant.h holds the formulas).
#include <algorithm>

#include "quant_common.cuh"
#include "quant_kernels.hpp"
#include "quant_launch.cuh"

namespace rns8cuda {
namespace {

constexpr int kMaxThreads = 1024;

struct Forward {
  int64_t rows_per_gate;
  int64_t ld_x, ld_y, ld_gate, ld_x_out, ld_h, ld_q;
  const void *x, *y, *post, *pre, *gate;
  void *x_out, *h;
  int8_t* q;
  float* q_scale;
  float scale, eps, offset, inv_dim;
  int dim;
};

// One block per token; the token's row stays in registers from its load to its
// stores.
template <typename T, typename W, bool ALIGNED, int NV>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_kernel(const Forward p) {
  __shared__ float slots[3][32];
  const int64_t t = blockIdx.x;
  const int n = blockDim.x, tid = threadIdx.x;
  wait_previous_launch();
  allow_next_launch();
  float y[NV][8], x[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load8<ALIGNED>(static_cast<const T*>(p.y) + t * p.ld_y, p.dim, j, n, tid, y[j]);
    load8<ALIGNED>(static_cast<const T*>(p.x) + t * p.ld_x, p.dim, j, n, tid, x[j]);
  }
  float f = p.scale;
  if (p.post) {
    float s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] += y[j][e] * y[j][e];
    block_sum(s, slots[0]);
    f *= rsqrtf(s[0] * p.inv_dim + p.eps);
  }
  float s[1] = {0.0f};
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float w[8], g[8];
    if (p.post) load8<ALIGNED>(static_cast<const W*>(p.post), p.dim, j, n, tid, w);
    if (p.gate) load8<ALIGNED>(static_cast<const W*>(p.gate) + t / p.rows_per_gate * p.ld_gate, p.dim, j, n, tid, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float u = y[j][e] * f;
      if (p.post) u *= p.offset + w[e];
      if (p.gate) u *= g[e];
      x[j][e] += u;
      s[0] += x[j][e] * x[j][e];
    }
    store8<ALIGNED>(static_cast<T*>(p.x_out) + t * p.ld_x_out, p.dim, j, n, tid, x[j]);
  }
  if (!p.pre) return;
  block_sum(s, slots[1]);
  const float rho = rsqrtf(s[0] * p.inv_dim + p.eps);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float w[8];
    load8<ALIGNED>(static_cast<const W*>(p.pre), p.dim, j, n, tid, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // Elements past the row are zero and stay zero whatever rho is: a row
      // that holds an infinity has rho = 0 or NaN, and its own elements say so.
      x[j][e] *= rho * (p.offset + w[e]);
      if (row_index<ALIGNED>(j, e, n, tid) < p.dim) top = max(top, magnitude_bits(x[j][e]));
    }
    if (p.h) store8<ALIGNED>(static_cast<T*>(p.h) + t * p.ld_h, p.dim, j, n, tid, x[j]);
  }
  if (!p.q) return;
  const RowScale rs = make_row_scale(block_max(top, reinterpret_cast<uint32_t*>(slots[2])));
  if (tid == 0) p.q_scale[t] = rs.scale;
#pragma unroll
  for (int j = 0; j < NV; ++j) store_q8<ALIGNED>(p.q + t * p.ld_q, p.dim, j, n, tid, x[j], rs.inv);
}

struct Backward {
  int64_t ld_dxo, ld_dh, ld_x, ld_y, ld_gate, ld_dx, ld_dy, ld_dgate;
  const void *dxo, *dh, *x, *y, *post, *pre, *gate;
  void *dx, *dy, *dgate;
  float *part_post, *part_pre, *part_gate;  // per-block sums [grid][dim], per-item gate sums [items][dim]
  int64_t items, chunks, rows_per_item, rows_per_group, rows_per_gate;
  float scale, eps, offset, inv_dim;
  int dim;
  bool per_token;  // one gate row per token: d_gate is written token by token
};

// A block walks items (runs of tokens that share a gate row) and keeps the
// sums over tokens in registers: for dgate and dpost A = sum of u * dx over an
// item (both are multiples of it by per-channel factors), for dpre its own.
// The row needs one reduction: with a = scale * gate * (offset + post),
// mean(v u) expands over dx = dxo + rho t - rho^2 mean(t n) x into sums that do
// not depend on dx.
template <typename T, typename W, bool ALIGNED, int NV>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_backward_kernel(const Backward p) {
  __shared__ float slots[2][6 * 32];
  const int n = blockDim.x, tid = threadIdx.x;
  wait_previous_launch();
  allow_next_launch();
  float acc_pre[NV][8] = {}, acc_post[NV][8] = {};
  int buf = 0;
  for (int64_t item = blockIdx.x; item < p.items; item += gridDim.x) {
    const int64_t group = item / p.chunks, first = group * p.rows_per_group + (item % p.chunks) * p.rows_per_item;
    const int64_t last = min(first + p.rows_per_item, (group + 1) * p.rows_per_group);
    float acc[NV][8] = {};
    for (int64_t t = first; t < last; ++t, buf ^= 1) {
      const T* dxo = p.dxo ? static_cast<const T*>(p.dxo) + t * p.ld_dxo : nullptr;
      const T* dh = p.dh ? static_cast<const T*>(p.dh) + t * p.ld_dh : nullptr;
      const T* x = static_cast<const T*>(p.x) + t * p.ld_x;
      const T* y = static_cast<const T*>(p.y) + t * p.ld_y;
      const W* gate = p.gate ? static_cast<const W*>(p.gate) + t / p.rows_per_gate * p.ld_gate : nullptr;
      struct Vec {
        float dxo[8], dh[8], x[8], y[8], a[8], g[8], w[8], pre[8];
      };
      auto load = [&](int j, Vec& v) {
        load8<ALIGNED>(x, p.dim, j, n, tid, v.x);
        load8<ALIGNED>(y, p.dim, j, n, tid, v.y);
        if (dxo) load8<ALIGNED>(dxo, p.dim, j, n, tid, v.dxo);
        if (dh) load8<ALIGNED>(dh, p.dim, j, n, tid, v.dh);
        if (p.pre) load8<ALIGNED>(static_cast<const W*>(p.pre), p.dim, j, n, tid, v.pre);
        if (p.post) load8<ALIGNED>(static_cast<const W*>(p.post), p.dim, j, n, tid, v.w);
        if (gate) load8<ALIGNED>(gate, p.dim, j, n, tid, v.g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (!dxo) v.dxo[e] = 0.0f;
          if (!dh) v.dh[e] = 0.0f;
          v.pre[e] = p.pre ? p.offset + v.pre[e] : 0.0f;
          v.w[e] = p.post ? p.offset + v.w[e] : 1.0f;
          v.g[e] = gate ? p.scale * v.g[e] : p.scale;
          v.a[e] = v.g[e] * v.w[e];
        }
      };
      Vec v0;
      float s[6] = {};
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        load(j, v0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float th = v0.dh[e] * v0.pre[e], ay = v0.a[e] * v0.y[e];
          s[0] += v0.x[e] * v0.x[e];
          s[1] += th * v0.x[e];
          s[2] += v0.y[e] * v0.y[e];
          s[3] += ay * v0.dxo[e];
          s[4] += ay * th;
          s[5] += ay * v0.x[e];
        }
      }
      block_sum(s, slots[buf]);
      const float rho = p.pre ? rsqrtf(s[0] * p.inv_dim + p.eps) : 0.0f;
      const float along = rho * rho * rho * s[1] * p.inv_dim;  // rho^2 mean(t n)
      const float sigma = p.post ? rsqrtf(s[2] * p.inv_dim + p.eps) : 1.0f;
      const float mvu = p.post ? sigma * (s[3] + rho * s[4] - along * s[5]) * p.inv_dim : 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (NV > 1) load(j, v0);
        float dx[8], dy[8], dg[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dx[e] = v0.dxo[e] + rho * (v0.dh[e] * v0.pre[e]) - along * v0.x[e];
          const float u = v0.y[e] * sigma;
          dy[e] = sigma * (v0.a[e] * dx[e] - u * mvu);
          acc_pre[j][e] += v0.dh[e] * (v0.x[e] * rho);
          const float udx = u * dx[e];
          if (p.per_token) {
            dg[e] = p.scale * v0.w[e] * udx;
            acc_post[j][e] += v0.g[e] * udx;
          } else {
            acc[j][e] += udx;
          }
        }
        store8<ALIGNED>(static_cast<T*>(p.dx) + t * p.ld_dx, p.dim, j, n, tid, dx);
        store8<ALIGNED>(static_cast<T*>(p.dy) + t * p.ld_dy, p.dim, j, n, tid, dy);
        if (p.per_token && p.dgate) store8<ALIGNED>(static_cast<T*>(p.dgate) + t * p.ld_dgate, p.dim, j, n, tid, dg);
      }
    }
    if (!p.per_token) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float w[8], g[8], dg[8];
        if (p.post) load8<ALIGNED>(static_cast<const W*>(p.post), p.dim, j, n, tid, w);
        if (p.gate) load8<ALIGNED>(static_cast<const W*>(p.gate) + first / p.rows_per_gate * p.ld_gate, p.dim, j, n, tid, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dg[e] = p.scale * (p.post ? p.offset + w[e] : 1.0f) * acc[j][e];
          acc_post[j][e] += (p.gate ? p.scale * g[e] : p.scale) * acc[j][e];
        }
        if (p.part_gate) {
          store8<ALIGNED>(p.part_gate + item * p.dim, p.dim, j, n, tid, dg);
        } else if (p.dgate) {
          float* out = static_cast<float*>(p.dgate) + group * p.ld_dgate;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = row_index<ALIGNED>(j, e, n, tid);
            if (i < p.dim) out[i] = dg[e];
          }
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (p.part_post) store8<ALIGNED>(p.part_post + static_cast<int64_t>(blockIdx.x) * p.dim, p.dim, j, n, tid, acc_post[j]);
    if (p.part_pre) store8<ALIGNED>(p.part_pre + static_cast<int64_t>(blockIdx.x) * p.dim, p.dim, j, n, tid, acc_pre[j]);
  }
}

// out[g][c] = sum over the group's `count` consecutive rows of part. A block
// sums 32 columns with 8 row lanes, always in the same order. blockIdx.z picks
// one of three sums.
struct Sums {
  const float* part[3];
  float* out[3];
  int64_t count[3], groups[3], ld_out[3];
  int dim;
};
__global__ void __launch_bounds__(256) sum_rows_kernel(const Sums p) {
  __shared__ float s[8][33];
  const int z = blockIdx.z;
  wait_previous_launch();
  allow_next_launch();
  if (!p.out[z]) return;
  const int c = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
  for (int64_t g = blockIdx.y; g < p.groups[z]; g += gridDim.y) {
    float v = 0.0f;
    if (c < p.dim)
      for (int64_t r = lane; r < p.count[z]; r += 8) v += p.part[z][(g * p.count[z] + r) * p.dim + c];
    s[lane][threadIdx.x % 32] = v;
    __syncthreads();
    if (lane == 0 && c < p.dim) {
      for (int i = 1; i < 8; ++i) v += s[i][threadIdx.x];
      p.out[z][g * p.ld_out[z] + c] = v;
    }
    __syncthreads();
  }
}

bool aligned_rows(const void* p, int64_t ld, size_t elem) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * elem % 16 == 0);
}
size_t type_size(uint32_t t) { return t == RNS8_CUDA_TYPE_F32 ? 4 : 2; }

unsigned block_threads(int dim, int nv) {
  return static_cast<unsigned>(std::max(32, (((dim + 7) / 8 + nv - 1) / nv + 31) / 32 * 32));
}

// Calls f(T, W, ALIGNED, NV) as types for the descriptor's element types.
template <typename F>
cudaError_t dispatch(uint32_t type, uint32_t weight_type, bool aligned, int nv, F&& f) {
  auto with = [&](auto t, auto w) {
    auto al = [&](auto a) {
      if (nv == 1) return f(t, w, a, std::integral_constant<int, 1>{});
      if (nv == 2) return f(t, w, a, std::integral_constant<int, 2>{});
      return f(t, w, a, std::integral_constant<int, 4>{});
    };
    return aligned ? al(std::true_type{}) : al(std::false_type{});
  };
  if (type == RNS8_CUDA_TYPE_F32) return with(float{}, float{});
  if (type == RNS8_CUDA_TYPE_BF16)
    return weight_type == RNS8_CUDA_TYPE_F32 ? with(__nv_bfloat16{}, float{}) : with(__nv_bfloat16{}, __nv_bfloat16{});
  return weight_type == RNS8_CUDA_TYPE_F32 ? with(__half{}, float{}) : with(__half{}, __half{});
}

// How the backward pass splits its tokens: items of one gate row each, at
// most `chunks` items per gate row, walked by `grid` blocks.
struct Split {
  int64_t groups, rows_per_group, chunks, rows_per_item, items;
  int64_t grid;
  bool per_token;
};
Split split_tokens(const rns8_cuda_residual_norm_backward_desc& d, int sm_count) {
  Split s;
  const int64_t target = 2 * static_cast<int64_t>(sm_count);
  s.per_token = d.gate && d.groups == d.tokens;
  s.groups = (s.per_token || !d.gate) ? 1 : d.groups;
  s.rows_per_group = d.tokens / s.groups;
  s.chunks = std::min(s.rows_per_group, (target + s.groups - 1) / s.groups);
  s.rows_per_item = (s.rows_per_group + s.chunks - 1) / s.chunks;
  s.chunks = (s.rows_per_group + s.rows_per_item - 1) / s.rows_per_item;
  s.items = s.groups * s.chunks;
  s.grid = std::min(s.items, target);
  return s;
}
bool gate_partials(const rns8_cuda_residual_norm_backward_desc& d, const Split& s) {
  return d.gate && d.d_gate && !s.per_token && s.chunks > 1;
}

}  // namespace

cudaError_t residual_norm(const rns8_cuda_residual_norm_desc& d, cudaStream_t stream) {
  Forward p{};
  p.rows_per_gate = d.gate ? d.tokens / d.groups : 1;
  p.ld_x = d.ld_x, p.ld_y = d.ld_y, p.ld_gate = d.ld_gate, p.ld_x_out = d.ld_x_out, p.ld_h = d.ld_h, p.ld_q = d.ld_q;
  p.x = d.x, p.y = d.y, p.post = d.post_weight, p.pre = d.pre_weight, p.gate = d.gate;
  p.x_out = d.x_out, p.h = d.h, p.q = d.q, p.q_scale = d.q_scale;
  p.scale = d.scale, p.eps = d.eps, p.offset = d.weight_offset, p.dim = static_cast<int>(d.dim);
  p.inv_dim = 1.0f / static_cast<float>(p.dim);
  const size_t e = type_size(d.type), w = type_size(d.weight_type);
  const bool aligned = aligned_rows(d.x, d.ld_x, e) && aligned_rows(d.y, d.ld_y, e) &&
                       aligned_rows(d.post_weight, 0, w) && aligned_rows(d.pre_weight, 0, w) &&
                       aligned_rows(d.gate, d.ld_gate, w) && aligned_rows(d.x_out, d.ld_x_out, e) &&
                       aligned_rows(d.h, d.ld_h, e) &&
                       (!d.q || (reinterpret_cast<uintptr_t>(d.q) % 8 == 0 && d.ld_q % 8 == 0));
  const int vectors = row_vectors(d.tokens, (p.dim + 7) / 8);
  return dispatch(d.type, d.weight_type, aligned, vectors, [&](auto t, auto wt, auto al, auto nv) {
    constexpr int NV = decltype(nv)::value;
    return launch_chained(residual_norm_kernel<decltype(t), decltype(wt), decltype(al)::value, NV>,
                          dim3(static_cast<unsigned>(d.tokens)), block_threads(p.dim, NV), 0, 1, stream, p);
  });
}

uint64_t residual_norm_backward_scratch_bytes(const rns8_cuda_residual_norm_backward_desc& d, int sm_count) {
  const Split s = split_tokens(d, sm_count);
  uint64_t rows = 0;
  if (d.d_post) rows += s.grid;
  if (d.d_pre) rows += s.grid;
  if (gate_partials(d, s)) rows += s.items;
  return rows * static_cast<uint64_t>(d.dim) * sizeof(float) + (rows ? 16 : 0);
}

cudaError_t residual_norm_backward(const rns8_cuda_residual_norm_backward_desc& d, int sm_count, cudaStream_t stream) {
  const Split s = split_tokens(d, sm_count);
  Backward p{};
  p.ld_dxo = d.ld_d_x_out, p.ld_dh = d.ld_d_h, p.ld_x = d.ld_x_out, p.ld_y = d.ld_y, p.ld_gate = d.ld_gate;
  p.ld_dx = d.ld_d_x, p.ld_dy = d.ld_d_y, p.ld_dgate = d.ld_d_gate;
  p.dxo = d.d_x_out, p.dh = d.pre_weight ? d.d_h : nullptr, p.x = d.x_out, p.y = d.y;
  p.post = d.post_weight, p.pre = d.pre_weight, p.gate = d.gate;
  p.dx = d.d_x, p.dy = d.d_y, p.dgate = d.gate ? d.d_gate : nullptr;
  p.items = s.items, p.chunks = s.chunks, p.rows_per_item = s.rows_per_item, p.rows_per_group = s.rows_per_group;
  p.rows_per_gate = d.gate ? d.tokens / d.groups : 1;
  p.per_token = s.per_token;
  p.scale = d.scale, p.eps = d.eps, p.offset = d.weight_offset, p.dim = static_cast<int>(d.dim);
  p.inv_dim = 1.0f / static_cast<float>(p.dim);

  float* next = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(d.scratch) + 15) & ~uintptr_t(15));
  auto take = [&](int64_t rows) {
    float* at = next;
    next += rows * d.dim;
    return at;
  };
  Sums sums{};
  sums.dim = p.dim;
  if (d.d_post) {
    p.part_post = take(s.grid);
    sums.part[0] = p.part_post, sums.out[0] = d.d_post, sums.count[0] = s.grid, sums.groups[0] = 1;
  }
  if (d.d_pre) {
    p.part_pre = take(s.grid);
    sums.part[1] = p.part_pre, sums.out[1] = d.d_pre, sums.count[1] = s.grid, sums.groups[1] = 1;
  }
  if (gate_partials(d, s)) {
    p.part_gate = take(s.items);
    sums.part[2] = p.part_gate, sums.out[2] = static_cast<float*>(d.d_gate);
    sums.count[2] = s.chunks, sums.groups[2] = s.groups, sums.ld_out[2] = d.ld_d_gate;
  }

  const size_t e = type_size(d.type), w = type_size(d.weight_type);
  const bool aligned = aligned_rows(d.d_x_out, d.ld_d_x_out, e) && aligned_rows(d.d_h, d.ld_d_h, e) &&
                       aligned_rows(d.x_out, d.ld_x_out, e) && aligned_rows(d.y, d.ld_y, e) &&
                       aligned_rows(d.post_weight, 0, w) && aligned_rows(d.pre_weight, 0, w) &&
                       aligned_rows(d.gate, d.ld_gate, w) && aligned_rows(d.d_x, d.ld_d_x, e) &&
                       aligned_rows(d.d_y, d.ld_d_y, e) && d.dim % 4 == 0 &&
                       (!s.per_token || aligned_rows(d.d_gate, d.ld_d_gate, e));
  const int vectors = (p.dim + 7) / 8 <= kMaxThreads ? 1 : 4;
  cudaError_t err = dispatch(d.type, d.weight_type, aligned, vectors, [&](auto t, auto wt, auto al, auto nv) {
    constexpr int NV = decltype(nv)::value;
    return launch_chained(residual_norm_backward_kernel<decltype(t), decltype(wt), decltype(al)::value, NV>,
                          dim3(static_cast<unsigned>(s.grid)), block_threads(p.dim, NV), 0, 1, stream, p);
  });
  if (err != cudaSuccess) return err;
  if (sums.out[0] || sums.out[1] || sums.out[2]) {
    const unsigned gy = static_cast<unsigned>(std::min<int64_t>(sums.out[2] ? s.groups : 1, 1024));
    err = launch_chained(sum_rows_kernel, dim3((p.dim + 31) / 32, gy, 3), 256, 0, 1, stream, sums);
  }
  return err;
}

}  // namespace rns8cuda
