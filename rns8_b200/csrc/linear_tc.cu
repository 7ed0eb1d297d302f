// Scaled int8 product on the tensor cores (tcgen05.mma kind::i8).
//
// Two forms, both with TMA rings of 128-byte spans of k (128-byte swizzle, both
// operands K-major), int32 accumulators in tensor memory and the scales, bias
// and gate applied on the way out:
//
//   tokens on lanes   A persistent kernel, one block per SM: 128 tokens x 256
//                     weight rows (gated: 128 gate rows and their 128 up rows)
//                     per tile, two accumulators, so that a tile's epilogue
//                     runs under the next tile's products. For products with
//                     about a tile per SM or more.
//   channels on lanes One tile of 128 weight rows (gated: 64 gate rows and
//                     their 64 up rows) x 16..256 tokens per cluster; the
//                     blocks of a cluster split k and join their exact integer
//                     sums through distributed shared memory. For the rest:
//                     few tokens, where the weights' stream bounds it, and
//                     shapes with fewer tiles than SMs.
//
// Every mbarrier wait is bounded (by wait_cycles, those before a block leaves by
// the full limit); one that runs out sets the device status word and the block
// drains its copies and products and exits.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "device_common.cuh"
#include "gemm_internal.hpp"
#include "linear_internal.hpp"
#include "quant_kernels.hpp"
#include "quant_common.cuh"
#include "quant_launch.cuh"

namespace rns8cuda {
namespace {

constexpr int BK = 128, UMMA_K = 32, LANES = 128, THREADS = 192;
constexpr int kMaxSplits = 8;  // blocks of a cluster
constexpr uint32_t SPAN_BYTES = LANES * BK;  // one 128-row operand tile of a stage

struct __align__(64) TcLinear {
  CUtensorMap tm_tokens, tm_weights;
  const float *a_scale, *w_scale, *bias;
  void* out;
  int64_t m, n, ld_out;
  uint32_t total_kb;
  uint32_t m_tiles, n_tiles, units;  // tokens on lanes
  uint32_t after_quantize, vector_rows;
  uint32_t* status;
  int64_t wait_cycles;
};

__device__ __forceinline__ void report_timeout(const TcLinear& p, volatile int* abort_flag) {
  *abort_flag = 1;
  atomicOr(p.status, kDevWaitTimeout);
}

// silu(g) * u. The quick division is within 2 ulp and gives 0 for a divisor past
// 2^126, where the quotient is below 2^-118 for any g that has one.
__device__ __forceinline__ float silu_times(float g, float u) { return __fdividef(g, 1.0f + expf(-g)) * u; }

// Barrier of a kernel's epilogue warps that also ands their predicates.
template <int EPILOGUE_THREADS>
__device__ __forceinline__ bool epilogue_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(ok ? 1u : 0u), "n"(EPILOGUE_THREADS)
      : "memory");
  return all != 0;
}

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Sixteen bytes of block `rank`'s shared memory.
__device__ __forceinline__ int4 ld_cluster(const void* smem_ptr, uint32_t rank) {
  uint32_t at;
  int4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(smem_ptr)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at));
  return v;
}

// Stores G tokens x 32 channels of a warp: lane l holds channel j0 + l of every
// token, the warp's slice of shared memory turns that into runs of 32 channels
// and each lane stores G consecutive channels of token l / (32 / G) as one
// word (a store of single elements a token costs some 50 cycles each).
// `wide`: whole words are aligned. Tokens from `tokens` on and channels from
// `channels` on are left out.
template <typename OUT, int G>
__device__ __forceinline__ void store_turned(OUT* __restrict__ out, int64_t ld, const float (&y)[G], OUT* slice,
                                             int lane, int tokens, int64_t channels, bool wide) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < G; ++i) slice[i * 32 + lane] = from_f32<OUT>(y[i]);
  __syncwarp();
  constexpr int LANES_PER_TOKEN = 32 / G;
  const int t = lane / LANES_PER_TOKEN, c = lane % LANES_PER_TOKEN * G;
  if (t >= tokens) return;
  OUT* to = out + t * ld + c;
  const OUT* from = slice + t * 32 + c;
  if (wide && c + G <= channels) {
    if constexpr (G * sizeof(OUT) == 8) {
      *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from);
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(G * sizeof(OUT) / 16); ++i)
        reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(from)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < G; ++i)
      if (c + i < channels) to[i] = from[i];
  }
}

// ---- channels on lanes -------------------------------------------------------------
template <int BN>
struct Lanes {
  static constexpr uint32_t STAGE = SPAN_BYTES + BN * BK;
  // Two blocks share an SM (one for 256 tokens): a block alone streams at no
  // more than half of an SM's share of HBM.
  static constexpr int PER_SM = BN <= 128 ? 2 : 1;
  static constexpr int STAGES = (PER_SM == 2 ? 104 * 1024 : 196 * 1024) / STAGE;
  static constexpr uint32_t TMEM_COLS = BN < 32 ? 32 : BN;
  // Epilogue warps, one or two for each quarter of the lanes (1024 x 1024,
  // k 1024: 256 tokens to a tile 9.4 us with four, 8.0 with eight; 16 tokens
  // 3.3 and 3.5).
  static constexpr int WARPS = BN <= 32 ? 4 : 8, THREADS = 64 + 32 * WARPS;
  static constexpr uint32_t TURN = 8 * 32 * 4;  // store_turned's slice of a warp
  static constexpr size_t SMEM = 1024 + STAGES * STAGE + 256 + BN * sizeof(float) + WARPS * TURN;
  static_assert(BN * LANES * 4 <= STAGES * STAGE, "the joined sums reuse the stages");
};

template <typename OUT, int BN, bool GATED>
__global__ void __launch_bounds__(Lanes<BN>::THREADS, Lanes<BN>::PER_SM) linear_channels_kernel(const __grid_constant__ TcLinear p) {
  using L = Lanes<BN>;
  constexpr int STAGES = L::STAGES, CHANNELS = GATED ? LANES / 2 : LANES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * L::STAGE);
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* token_scale = reinterpret_cast<float*>(smem + STAGES * L::STAGE + 256);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  uint32_t rank, splits;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  // Clusters of one channel tile follow one another: they share its weights in L2.
  const int64_t j0 = static_cast<int64_t>(blockIdx.y) * CHANNELS, t0 = static_cast<int64_t>(blockIdx.x / splits) * BN;
  const uint32_t kb0 = p.total_kb * rank / splits, kb1 = p.total_kb * (rank + 1) / splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&p.tm_weights);
    tma_prefetch_desc(&p.tm_tokens);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // After this call's own quantisation the weights are not waited for: that
  // kernel has seen everything before it complete.
  if (!p.after_quantize) wait_previous_launch();
  allow_next_launch();

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer ----------------
      auto load_weights = [&](uint32_t stage, uint32_t kb) {
        uint8_t* at = smem + stage * L::STAGE;
        mbar_arrive_expect_tx(&full[stage], L::STAGE);
        tma_load_2d(at, &p.tm_weights, &full[stage], static_cast<int32_t>(kb * BK), static_cast<int32_t>(j0));
        if (GATED)
          tma_load_2d(at + SPAN_BYTES / 2, &p.tm_weights, &full[stage], static_cast<int32_t>(kb * BK),
                      static_cast<int32_t>(p.n + j0));
      };
      auto load_tokens = [&](uint32_t stage, uint32_t kb) {
        tma_load_2d(smem + stage * L::STAGE + SPAN_BYTES, &p.tm_tokens, &full[stage], static_cast<int32_t>(kb * BK),
                    static_cast<int32_t>(t0));
      };
      // The first stages' weights do not wait for the tokens to be quantised.
      const uint32_t early = min(kb1 - kb0, static_cast<uint32_t>(STAGES));
      for (uint32_t i = 0; i < early; ++i) load_weights(i, kb0 + i);
      if (p.after_quantize) wait_previous_launch();
      for (uint32_t i = 0; i < early; ++i) load_tokens(i, kb0 + i);
      uint32_t pending = (1u << early) - 1, parities = 0, stage = early % STAGES, phase = early / STAGES;
      for (uint32_t kb = kb0 + early; kb < kb1; ++kb) {
        if (*abort_flag || !mbar_wait_bounded(&empty[stage], phase ^ 1u, p.wait_cycles)) {
          if (!*abort_flag) report_timeout(p, abort_flag);
          break;
        }
        load_weights(stage, kb);
        load_tokens(stage, kb);
        pending |= 1u << stage;
        parities = (parities & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // Every copy has landed before the block may exit.
      for (int s = 0; s < STAGES; ++s)
        if (pending & (1u << s)) (void)mbar_wait_bounded(&full[s], (parities >> s) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t idesc = make_idesc_i8(LANES, BN, /*b_mn_major=*/false);
      uint32_t stage = 0, phase = 0;
      for (uint32_t kb = kb0; kb < kb1; ++kb) {
        if (*abort_flag || !mbar_wait_bounded(&full[stage], phase, p.wait_cycles)) {
          if (!*abort_flag) report_timeout(p, abort_flag);
          break;
        }
        tc_fence_after();
        const uint32_t sw = smem_u32(smem + stage * L::STAGE), st = sw + SPAN_BYTES;
#pragma unroll
        for (int kk = 0; kk < BK / UMMA_K; ++kk)
          tc_mma_i8(tmem_base, make_smem_desc_sw128(sw + kk * UMMA_K, 16, 1024),
                    make_smem_desc_sw128(st + kk * UMMA_K, 16, 1024), idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
        tc_commit(&empty[stage]);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      tc_commit(done);
      (void)mbar_wait_bounded(done, 0);
    }
  } else {
    // ---------------- epilogue (the other warps), first part ----------------
    if (p.after_quantize) wait_previous_launch();
    for (int c = threadIdx.x - 64; c < BN; c += 32 * L::WARPS) token_scale[c] = t0 + c < p.m ? p.a_scale[t0 + c] : 0.0f;
  }

  // A thread of the epilogue owns a channel: in the direct form (an ungated
  // tile of one block) its accumulator lane, else a lane of the joined sums,
  // where a gated tile has half as many and splits the tokens over its warps.
  const int quarter = warp & 3, ew = (warp - 2) & (L::WARPS - 1), cw = GATED ? quarter & 1 : quarter;
  const int64_t w0 = j0 + cw * 32, j = w0 + lane;  // the warp's first channel, this thread's
  const int tokens = static_cast<int>(min(p.m - t0, static_cast<int64_t>(BN)));
  OUT* out = static_cast<OUT*>(p.out) + t0 * p.ld_out + w0;
  OUT* slice = reinterpret_cast<OUT*>(reinterpret_cast<uint8_t*>(token_scale + BN) + ew * L::TURN);
  float ws = 0.0f, bias = 0.0f, up_ws = 0.0f, up_bias = 0.0f;
  if (warp >= 2 && j < p.n) {
    ws = p.w_scale[j];
    if (p.bias) bias = p.bias[j];
    if (GATED) {
      up_ws = p.w_scale[p.n + j];
      if (p.bias) up_bias = p.bias[p.n + j];
    }
  }
  auto value = [&](int c, int acc, int up) {
    const float s = token_scale[c];
    const float y = static_cast<float>(acc) * s * ws + bias;
    return GATED ? silu_times(y, static_cast<float>(up) * s * up_ws + up_bias) : y;
  };
  const bool direct = !GATED && splits == 1;
  int4* sums = reinterpret_cast<int4*>(smem);  // [BN / 4][LANES], once the stages are consumed
  if (warp >= 2) {
    if (!mbar_wait_bounded(done, 0, p.wait_cycles) && !*abort_flag) report_timeout(p, abort_flag);
    (void)epilogue_all<32 * L::WARPS>(true);  // the token scales are in place
    tc_fence_after();
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
    for (int c = ew / 4 * 32; c < tokens; c += L::WARPS * 8) {
      uint32_t v[32];
      __syncwarp();
      tmem_ld_32x32b_x32(taddr + c, v);
      tmem_wait_ld(v);
#pragma unroll
      for (int i = 0; i < (BN < 32 ? BN : 32); i += 8) {
        if (direct) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = value(c + i + e, static_cast<int>(v[i + e]), 0);
          store_turned<OUT, 8>(out + (c + i) * p.ld_out, p.ld_out, y, slice, lane, tokens - c - i, p.n - w0,
                               p.vector_rows);
        } else {
#pragma unroll
          for (int e = i; e < i + 8; e += 4)
            sums[((c + e) / 4) * LANES + quarter * 32 + lane] =
                make_int4(static_cast<int>(v[e]), static_cast<int>(v[e + 1]), static_cast<int>(v[e + 2]),
                          static_cast<int>(v[e + 3]));
        }
      }
    }
  }
  if (!direct) {
    // Each block of the cluster joins a share of the tile's tokens, four at a
    // time; all the blocks' parts of the next four are on their way meanwhile.
    cluster_sync();
    if (warp >= 2) {
      constexpr int WARPS_PER_TOKEN = CHANNELS / 32, SHARES = L::WARPS / WARPS_PER_TOKEN, PARTS = GATED ? 2 : 1;
      const int share = GATED ? (ew / 4) * 2 + quarter / 2 : ew / 4, step = 4 * static_cast<int>(splits) * SHARES;
      int4 next[PARTS][kMaxSplits];
      auto fetch = [&](int c) {
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r)
#pragma unroll
          for (int h = 0; h < PARTS; ++h)
            next[h][r] = r < static_cast<int>(splits)
                             ? ld_cluster(&sums[(c / 4) * LANES + h * CHANNELS + cw * 32 + lane], r)
                             : make_int4(0, 0, 0, 0);
      };
      int c = 4 * (static_cast<int>(rank) * SHARES + share);
      if (c < tokens) fetch(c);
      for (; c < tokens; c += step) {
        int4 total[PARTS];
#pragma unroll
        for (int h = 0; h < PARTS; ++h) {
          total[h] = next[h][0];
#pragma unroll
          for (int r = 1; r < kMaxSplits; ++r) {
            total[h].x += next[h][r].x;
            total[h].y += next[h][r].y;
            total[h].z += next[h][r].z;
            total[h].w += next[h][r].w;
          }
        }
        if (c + step < tokens) fetch(c + step);
        const int4 a = total[0], u = total[PARTS - 1];
        const float y[4] = {value(c, a.x, u.x), value(c + 1, a.y, u.y), value(c + 2, a.z, u.z), value(c + 3, a.w, u.w)};
        store_turned<OUT, 4>(out + c * p.ld_out, p.ld_out, y, slice, lane, tokens - c, p.n - w0, p.vector_rows);
      }
    }
    cluster_sync();  // no block leaves while another reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::TMEM_COLS);
  }
}

// ---- tokens on lanes ----------------------------------------------------------------
constexpr int BN = 256, STAGES = 4, GROUP_M = 32;
constexpr uint32_t STAGE_BYTES = SPAN_BYTES + BN * BK;
constexpr size_t TOKENS_SMEM = 1024 + STAGES * STAGE_BYTES + 256 + 2 * 2 * BN * sizeof(float);

template <typename OUT, bool GATED>
__global__ void __launch_bounds__(THREADS, 1) linear_tokens_kernel(const __grid_constant__ TcLinear p) {
  constexpr int COLS = GATED ? BN / 2 : BN;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* col_scale = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES + 256);  // [2][BN]
  float* col_bias = col_scale + 2 * BN;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 128);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&p.tm_weights);
    tma_prefetch_desc(&p.tm_tokens);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_previous_launch();
  allow_next_launch();

  // Tiles run down columns of GROUP_M token tiles, so that the tiles in flight
  // share operands in L2.
  auto tile_of = [&](uint32_t u, uint32_t& mt, uint32_t& nt) {
    const uint32_t span = GROUP_M * p.n_tiles, group = u / span, in = u - group * span;
    const uint32_t size = min(p.m_tiles - group * GROUP_M, static_cast<uint32_t>(GROUP_M));
    mt = group * GROUP_M + in % size;
    nt = in / size;
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, pending = 0, parities = 0;
      bool ok = true;
      for (uint32_t u = blockIdx.x; ok && u < p.units; u += gridDim.x) {
        uint32_t mt, nt;
        tile_of(u, mt, nt);
        const int32_t w0 = static_cast<int32_t>(nt * COLS);
        const int32_t w1 = GATED ? static_cast<int32_t>(p.n + nt * COLS) : w0 + BN / 2;
        for (uint32_t kb = 0; kb < p.total_kb; ++kb) {
          if (*abort_flag || !mbar_wait_bounded(&empty[stage], phase ^ 1u, p.wait_cycles)) {
            if (!*abort_flag) report_timeout(p, abort_flag);
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[stage], STAGE_BYTES);
          uint8_t* at = smem + stage * STAGE_BYTES;
          const int32_t k = static_cast<int32_t>(kb * BK);
          tma_load_2d(at, &p.tm_tokens, &full[stage], k, static_cast<int32_t>(mt * LANES));
          tma_load_2d(at + SPAN_BYTES, &p.tm_weights, &full[stage], k, w0);
          tma_load_2d(at + 2 * SPAN_BYTES, &p.tm_weights, &full[stage], k, w1);
          pending |= 1u << stage;
          parities = (parities & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      for (int s = 0; s < STAGES; ++s)
        if (pending & (1u << s)) (void)mbar_wait_bounded(&full[s], (parities >> s) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_i8(LANES, BN, /*b_mn_major=*/false);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (uint32_t u = blockIdx.x; ok && u < p.units; u += gridDim.x) {
        if (*abort_flag || !mbar_wait_bounded(&acc_empty[acc], acc_phase ^ 1u, p.wait_cycles)) {
          if (!*abort_flag) report_timeout(p, abort_flag);
          break;
        }
        tc_fence_after();
        for (uint32_t kb = 0; kb < p.total_kb; ++kb) {
          if (*abort_flag || !mbar_wait_bounded(&full[stage], phase, p.wait_cycles)) {
            if (!*abort_flag) report_timeout(p, abort_flag);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * STAGE_BYTES), sb = sa + SPAN_BYTES;
#pragma unroll
          for (int kk = 0; kk < BK / UMMA_K; ++kk)
            tc_mma_i8(tmem_base + acc * BN, make_smem_desc_sw128(sa + kk * UMMA_K, 16, 1024),
                      make_smem_desc_sw128(sb + kk * UMMA_K, 16, 1024), idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          tc_commit(&empty[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit(&acc_full[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      tc_commit(drain);
      (void)mbar_wait_bounded(drain, 0);
    }
  } else {
    // ---------------- epilogue: a thread owns a token ----------------
    const uint32_t quarter = static_cast<uint32_t>(warp & 3);
    const int et = threadIdx.x - 64;
    uint32_t acc = 0, acc_phase = 0;
    for (uint32_t u = blockIdx.x; u < p.units; u += gridDim.x) {
      uint32_t mt, nt;
      tile_of(u, mt, nt);
      const int64_t n0 = static_cast<int64_t>(nt) * COLS;
      // The tile's column scales and biases, as laid out in the accumulator.
      float* cs = col_scale + acc * BN;
      float* cb = col_bias + acc * BN;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = et + i * 128;
        const int64_t col = n0 + (GATED ? et : c);
        const bool in = col < p.n;
        const int64_t w = GATED ? i * p.n + col : col;
        cs[c] = in ? p.w_scale[w] : 0.0f;
        cb[c] = in && p.bias ? p.bias[w] : 0.0f;
      }
      const int64_t t = static_cast<int64_t>(mt) * LANES + quarter * 32 + lane;
      const bool token = t < p.m;
      const float s = token ? p.a_scale[t] : 0.0f;
      const bool ok = !*abort_flag && mbar_wait_bounded(&acc_full[acc], acc_phase, p.wait_cycles);
      if (!ok && !*abort_flag) report_timeout(p, abort_flag);
      // The column values are in place, and the four warps stop together or
      // not at all: the next tile's barrier needs all of them.
      if (!epilogue_all<128>(ok)) break;
      tc_fence_after();
      OUT* orow = static_cast<OUT*>(p.out) + t * p.ld_out + n0;
      const uint32_t taddr = tmem_base + ((quarter * 32u) << 16) + acc * BN;
#pragma unroll 1
      for (int c = 0; c < COLS; c += 32) {
        uint32_t v[32], up[32];
        __syncwarp();
        tmem_ld_32x32b_x32(taddr + c, v);
        if (GATED) tmem_ld_32x32b_x32(taddr + BN / 2 + c, up);
        tmem_wait_ld(v);
        if (GATED) tmem_wait_ld(up);
        if (!token || n0 + c >= p.n) continue;
        __align__(16) OUT o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float y = static_cast<float>(static_cast<int>(v[i])) * s * cs[c + i] + cb[c + i];
          if (GATED)
            y = silu_times(y, static_cast<float>(static_cast<int>(up[i])) * s * cs[BN / 2 + c + i] + cb[BN / 2 + c + i]);
          o[i] = from_f32<OUT>(y);
        }
        if (p.vector_rows && n0 + c + 32 <= p.n) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(sizeof(o) / 16); ++i)
            reinterpret_cast<uint4*>(orow + c)[i] = reinterpret_cast<const uint4*>(o)[i];
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (n0 + c + i < p.n) orow[c + i] = o[i];
        }
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// ---- launches --------------------------------------------------------------------------
template <typename Kernel>
cudaError_t launch(Kernel kernel, std::atomic<uint64_t>& configured, dim3 grid, unsigned threads, unsigned cluster,
                   size_t smem, const TcLinear& p, cudaStream_t stream) {
  const cudaError_t e = raise_smem_limit_once(kernel, static_cast<int>(smem), configured);
  if (e != cudaSuccess) return e;
  return launch_chained(kernel, grid, threads, smem, cluster, stream, p);
}

template <typename OUT, int N, bool GATED>
cudaError_t launch_channels(const TcLinear& p, dim3 grid, unsigned splits, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  return launch(linear_channels_kernel<OUT, N, GATED>, configured, grid, Lanes<N>::THREADS, splits, Lanes<N>::SMEM, p,
                stream);
}
template <typename OUT, bool GATED>
cudaError_t launch_tokens(const TcLinear& p, unsigned grid, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  return launch(linear_tokens_kernel<OUT, GATED>, configured, dim3(grid), THREADS, 1, TOKENS_SMEM, p, stream);
}

template <typename F>
cudaError_t with_type(uint32_t type, F&& f) {
  if (type == RNS8_CUDA_TYPE_BF16) return f(__nv_bfloat16{});
  if (type == RNS8_CUDA_TYPE_F16) return f(__half{});
  return f(float{});
}

// Which form, tile and split a product runs, by an estimate of its time in us.
// With spans of 128 bytes of k, a block streams one in 0.12 us + its bytes at
// 155 GB/s when it has its SM to itself, at 75 GB/s beside another one; what a
// tile costs besides grows with its tokens, more when blocks join their sums,
// less the more of them share that; HBM gives the weights at 6.3 TB/s, less
// when several token tiles ask for them or when one block an SM does. Blocks
// that join wait for one another, so they are kept to one wave, with a tenth of
// the SMs to spare (a cluster needs its blocks free in one place).
// The constants are fitted to sweeps of both forms over 1 to 3000 tokens, 512
// to 8192 channels and k. Some of them, in us, as tokens to a tile / blocks to a
// cluster: 64 tokens 4096 x 4096: 8.4 as 64/4, 9.8 as 64/8, 12.0 as 16/1; 256
// tokens: 11.7 as 64/2, 14.5 as 256/2, 17.3 tokens on lanes; 700 tokens 8192 x
// 8192: 51.5 tokens on lanes, 57 as 128/1, 61 as 128/2.
struct Choice {
  bool tokens_on_lanes;
  int tile;
  unsigned splits;
  double us;
};
Choice choose(int64_t m, int64_t n, int64_t total_kb, bool gated, int sm_count) {
  const double weight_us = static_cast<double>(gated ? 2 * n : n) * total_kb * BK / 6.3e6;
  const double sms = sm_count;
  auto ceil_div = [](double a, double b) { return std::ceil(a / b); };
  const double units = ceil_div(m, LANES) * ceil_div(n, gated ? BN / 2 : BN);
  Choice best{true, 0, 1, 4.2 + std::max(weight_us, ceil_div(units, sms) * total_kb * 0.43)};
  const double channel_tiles = ceil_div(n, gated ? LANES / 2 : LANES);
  if (channel_tiles > 65535) return best;  // the grid's y extent
  for (int tile = 16; tile <= 256; tile *= 2) {
    const double token_tiles = ceil_div(m, tile), tiles = token_tiles * channel_tiles;
    const int per_sm = tile <= 128 ? 2 : 1;
    const double bytes = (LANES + tile) * BK * 1e-3, hbm = weight_us * (1 + 0.1 * (std::min(token_tiles, 5.0) - 1));
    for (unsigned splits = 1; splits <= kMaxSplits && (splits == 1 || total_kb >= 2 * splits); splits *= 2) {
      const double blocks = tiles * splits, waves = ceil_div(blocks, per_sm * sms);
      const bool shared = per_sm == 2 && blocks > sms;
      if (splits > 1 && blocks > 0.9 * per_sm * sms) break;
      const double span = shared ? bytes / 75 : 0.12 + bytes / 155;
      double rest = 0.1 + 0.011 * tile + 0.02 * tile / splits;
      if (shared) rest = 1.6 * rest + (splits == kMaxSplits ? 1.5 : 0.0);
      if (splits == 1 && !gated) rest = 0.005 * tile;
      const double us = 2.9 + waves * rest + std::max(shared ? hbm : 1.07 * hbm, waves * ceil_div(total_kb, splits) * span);
      if (us < best.us) best = Choice{false, tile, splits, us};
    }
    if (tile >= m) break;
  }
  return best;
}

}  // namespace

LinearForm linear_form(const rns8_cuda_linear_desc& d, int sm_count) {
  const Choice c = choose(d.m, d.n, (d.k + BK - 1) / BK, (d.flags & RNS8_CUDA_LINEAR_GATED) != 0, sm_count);
  return LinearForm{c.tokens_on_lanes ? 0u : static_cast<uint32_t>(c.tile), c.splits};
}

cudaError_t linear_tc(const LinearArgs& a, int sm_count, cudaStream_t stream) {
  TcLinear p{};
  p.a_scale = a.a_scale, p.w_scale = a.w_scale, p.bias = a.bias, p.out = a.out;
  p.m = a.m, p.n = a.n, p.ld_out = a.ld_out;
  p.total_kb = static_cast<uint32_t>((a.k + BK - 1) / BK);
  p.after_quantize = a.after_quantize;
  p.status = a.status;
  p.wait_cycles = quant_wait_cycles();
  const size_t elem = a.out_type == RNS8_CUDA_TYPE_F32 ? 4 : 2;
  p.vector_rows = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.ld_out * elem % 16 == 0;
  const int64_t w_rows = a.gated ? 2 * a.n : a.n;
  const Choice c = choose(a.m, a.n, p.total_kb, a.gated, sm_count);

  if (c.tokens_on_lanes) {
    const int cols = a.gated ? BN / 2 : BN;
    const uint64_t m_tiles = (a.m + LANES - 1) / LANES, n_tiles = (a.n + cols - 1) / cols;
    if (m_tiles * n_tiles >= (1ull << 32)) return cudaErrorInvalidValue;
    if (!encode_rows_i8(&p.tm_weights, a.w, w_rows, a.k, a.ld_w, LANES) ||
        !encode_rows_i8(&p.tm_tokens, a.a, a.m, a.k, a.ld_a, LANES))
      return cudaErrorInvalidValue;
    p.m_tiles = static_cast<uint32_t>(m_tiles);
    p.n_tiles = static_cast<uint32_t>(n_tiles);
    p.units = p.m_tiles * p.n_tiles;
    const unsigned grid = std::min<unsigned>(p.units, static_cast<unsigned>(sm_count));
    return with_type(a.out_type, [&](auto t) {
      using OUT = decltype(t);
      return a.gated ? launch_tokens<OUT, true>(p, grid, stream) : launch_tokens<OUT, false>(p, grid, stream);
    });
  }

  const int channels = a.gated ? LANES / 2 : LANES;
  if (!encode_rows_i8(&p.tm_weights, a.w, w_rows, a.k, a.ld_w, static_cast<uint32_t>(channels)) ||
      !encode_rows_i8(&p.tm_tokens, a.a, a.m, a.k, a.ld_a, static_cast<uint32_t>(c.tile)))
    return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>((a.m + c.tile - 1) / c.tile * c.splits),
                  static_cast<unsigned>((a.n + channels - 1) / channels));
  return with_type(a.out_type, [&](auto t) {
    using OUT = decltype(t);
    auto go = [&](auto g) {
      constexpr bool G = decltype(g)::value;
      switch (c.tile) {
        case 16: return launch_channels<OUT, 16, G>(p, grid, c.splits, stream);
        case 32: return launch_channels<OUT, 32, G>(p, grid, c.splits, stream);
        case 64: return launch_channels<OUT, 64, G>(p, grid, c.splits, stream);
        case 128: return launch_channels<OUT, 128, G>(p, grid, c.splits, stream);
        default: return launch_channels<OUT, 256, G>(p, grid, c.splits, stream);
      }
    };
    return a.gated ? go(std::true_type{}) : go(std::false_type{});
  });
}

}  // namespace rns8cuda
