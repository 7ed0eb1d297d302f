// The norms around a block fused with its gate and residual update, forward
// and backward (include/rns8/rns8_quant.h holds the formulas).
//
// Both directions move a few bytes per element and do some tens of operations
// on it, so HBM is to bound them; what stands in the way is that a row must be
// reduced before any of it can be written. Two forms each:
//
//   streamed  For many tokens: persistent blocks whose rows arrive in shared
//             memory through a ring of bulk copies, so that the next tokens'
//             bytes are on their way while this token is reduced.
//   direct    For few tokens, for very wide rows, and forward for rows that do
//             not start on 16-byte boundaries: a row read straight into
//             registers.
#include <algorithm>
#include <atomic>

#include "device_common.cuh"
#include "quant_common.cuh"
#include "quant_kernels.hpp"
#include "quant_launch.cuh"

namespace rns8cuda {
namespace {

constexpr int kMaxThreads = 1024;
static_assert(kQuantWaitCycles == kWaitBudgetCycles, "the limit that the kernels' last waits keep");

struct Forward {
  int64_t rows_per_gate;
  int64_t ld_x, ld_y, ld_gate, ld_x_out, ld_h, ld_q;
  const void *x, *y, *post, *pre, *gate;
  void *x_out, *h;
  int8_t* q;
  float* q_scale;
  float scale, eps, offset, inv_dim;
  int dim;
  bool q_words;
  int64_t wait_cycles;
};

// How a kernel reads and writes rows.
//   Words     On 16-byte boundaries, the width a multiple of 8.
//   Shifted   The rest (odd widths, slices): vectors shifted into place (4000 x
//             8191 bf16 98 us, element by element 203; 1 x 1001 2.7 and 4.0).
//   Elements  The rest where a vector a thread holds a row of floats (2000 x
//             1001 9.2 us, shifted 10.7; wider ones 249 and 171 at 8000 x 5001)
//             and in the streamed backward form: shared memory reads any
//             alignment alike, and shifting four rows costs more issue (4000 x
//             8191 f32 198 us, shifted 250).
enum class Access { Words, Shifted, Elements };

// Index of element e of this thread's vector j.
template <Access A>
__device__ __forceinline__ int element_index(int j, int e, int n, int tid) {
  return row_index<A != Access::Elements>(j, e, n, tid);
}
// Vector j of this thread's part of a row; elements at or past dim are zero.
template <Access A, typename T>
__device__ __forceinline__ Raw8<T> load_raw(const T* row, int dim, int j, int n, int tid) {
  if constexpr (A == Access::Words) {
    const int i = (j * n + tid) * 8;
    Raw8<T> v;
    v.load(row + i, i < dim);
    return v;
  } else if constexpr (A == Access::Shifted) {
    return load_shifted<T>(row, dim, (j * n + tid) * 8);
  } else {
    F2 v[4];
    load8<false>(row, dim, j, n, tid, v);
    Raw8<T> raw;
    raw.set(v);
    return raw;
  }
}
template <Access A, typename T>
__device__ __forceinline__ void load_row(const T* row, int dim, int j, int n, int tid, F2 (&v)[4]) {
  if constexpr (A == Access::Elements) {
    load8<false>(row, dim, j, n, tid, v);
  } else {
    const Raw8<T> raw = load_raw<A>(row, dim, j, n, tid);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = raw.pair(e);
  }
}
template <Access A, typename T>
__device__ __forceinline__ void store_row(T* row, int dim, int j, int n, int tid, const F2 (&v)[4]) {
  if constexpr (A == Access::Shifted) {
    Raw8<T> raw;
    raw.set(v);
    store_shifted<T>(row, dim, (j * n + tid) * 8, raw);
  } else {
    store8<A == Access::Words>(row, dim, j, n, tid, v);
  }
}
// Rows of partial sums, padded to whole vectors.
template <Access A>
__device__ __forceinline__ void store_partial(float* row, int dim, int j, int n, int tid, const F2 (&v)[4]) {
  store8<A != Access::Elements>(row, dim, j, n, tid, v);
}
// int8 values of a vector; q_words: q's rows are on 8-byte boundaries.
template <Access A>
__device__ __forceinline__ void store_row_q8(int8_t* row, bool q_words, int dim, int j, int n, int tid,
                                             const F2 (&v)[4], float inv) {
  if (A == Access::Words || (A == Access::Shifted && q_words && (j * n + tid) * 8 + 8 <= dim)) {
    store_q8<true>(row, dim, j, n, tid, v, inv);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = element_index<A>(j, e, n, tid);
      if (i < dim) row[i] = static_cast<int8_t>(quantize_one(e % 2 ? v[e / 2].v.y : v[e / 2].v.x, inv));
    }
  }
}

// Sum of a row's squares over the block.
template <int NV>
__device__ __forceinline__ float row_squares(const F2 (&v)[NV][4], SumSlots<1>& slots) {
  F2 s = f2(0.0f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fma(v[j][e], v[j][e], s);
  float sum[1] = {both(s)};
  block_sum(sum, slots);
  return sum[0];
}

// x += f * y * (offset + post) * gate for one vector; f holds scale and y's row
// factor. The options' branches are taken per vector.
template <Access A, typename T, typename W>
__device__ __forceinline__ void add_update(const Forward& p, const W* gate, float f, int j, int n, int tid,
                                           const F2 (&y)[4], F2 (&x)[4]) {
  F2 m[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) m[e] = f2(f);
  if (p.post) {
    F2 w[4];
    load_row<A>(static_cast<const W*>(p.post), p.dim, j, n, tid, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = m[e] * (w[e] + f2(p.offset));
  }
  if (p.gate) {
    F2 g[4];
    load_row<A>(gate, p.dim, j, n, tid, g);
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = m[e] * g[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = fma(y[e], m[e], x[e]);
}
template <Access A, typename W>
__device__ __forceinline__ void normalize(const Forward& p, float rho, int j, int n, int tid, F2 (&x)[4]) {
  F2 w[4];
  load_row<A>(static_cast<const W*>(p.pre), p.dim, j, n, tid, w);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = x[e] * (f2(rho) * (w[e] + f2(p.offset)));
}
// Largest magnitude of a vector. Elements past the row are left out: they are
// zero, but a row that holds an infinity has rho = 0 or NaN.
template <Access A>
__device__ __forceinline__ uint32_t row_magnitude(const F2 (&v)[4], int dim, int j, int n, int tid) {
  if (A == Access::Words) return (j * n + tid) * 8 < dim ? magnitude_bits(v) : 0u;
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (element_index<A>(j, e, n, tid) < dim) top = max(top, magnitude_bits(e % 2 ? v[e / 2].v.y : v[e / 2].v.x));
  return top;
}

// One block per token; the token's row stays in registers from its load to its
// stores.
template <typename T, typename W, Access A, int NV>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_kernel(const Forward p) {
  __shared__ SumSlots<1> slots[2];
  __shared__ uint32_t max_slots[32];
  const int64_t t = blockIdx.x;
  const int n = blockDim.x, tid = threadIdx.x;
  clear_slots(slots[0]);
  clear_slots(slots[1]);
  __syncthreads();
  wait_previous_launch();
  allow_next_launch();
  F2 y[NV][4], x[NV][4];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load_row<A>(static_cast<const T*>(p.y) + t * p.ld_y, p.dim, j, n, tid, y[j]);
    load_row<A>(static_cast<const T*>(p.x) + t * p.ld_x, p.dim, j, n, tid, x[j]);
  }
  const W* gate = static_cast<const W*>(p.gate) + (p.gate ? t / p.rows_per_gate * p.ld_gate : 0);
  float f = p.scale;
  if (p.post) f *= rsqrtf(row_squares(y, slots[0]) * p.inv_dim + p.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    add_update<A, T, W>(p, gate, f, j, n, tid, y[j], x[j]);
    store_row<A>(static_cast<T*>(p.x_out) + t * p.ld_x_out, p.dim, j, n, tid, x[j]);
  }
  if (!p.pre) return;
  const float rho = rsqrtf(row_squares(x, slots[1]) * p.inv_dim + p.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    normalize<A, W>(p, rho, j, n, tid, x[j]);
    if (p.h) store_row<A>(static_cast<T*>(p.h) + t * p.ld_h, p.dim, j, n, tid, x[j]);
  }
  if (!p.q) return;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) top = max(top, row_magnitude<A>(x[j], p.dim, j, n, tid));
  const RowScale rs = make_row_scale(block_max(top, max_slots));
  if (tid == 0) p.q_scale[t] = rs.scale;
#pragma unroll
  for (int j = 0; j < NV; ++j) store_row_q8<A>(p.q + t * p.ld_q, p.q_words, p.dim, j, n, tid, x[j], rs.inv);
}

// ---- rows through shared memory -----------------------------------------------------
constexpr int kMaxRing = 8;

// Room for a row, or for the 16-byte words around one that starts anywhere.
__host__ __device__ constexpr uint32_t row_room(bool aligned, int dim, uint32_t elem) {
  return aligned ? dim * elem : (dim * elem + 15) / 16 * 16 + 16;
}
__device__ __forceinline__ uint32_t row_offset(const void* row) { return reinterpret_cast<uintptr_t>(row) % 16; }
// Whether a token's rows are copied: the words around the first and the last
// may reach outside their matrices (those of the rows between do not, with rows
// of at least one word). Such tokens are read from global memory.
template <Access A>
__device__ __forceinline__ bool copied(int64_t t, int64_t tokens) {
  return A == Access::Words || (t > 0 && t < tokens - 1);
}

// Asks for whole 16-byte words of global memory to be brought into L2.
__device__ __forceinline__ void prefetch_l2(const void* words, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(words), "r"(bytes) : "memory");
}

// A ring of `stages` slots, each room for ROWS rows, filled by one thread's bulk
// copies of the 16-byte words around them. A wait that runs out cannot be reported (these calls
// have no status word), so it does not change the result instead: the thread
// reads its part of that and every later row from global memory.
template <int ROWS>
struct RowRing {
  uint8_t* base;
  uint64_t* full;
  uint32_t row_bytes, room, stages;
  int64_t wait_cycles;
  uint32_t stage = 0, phase = 0;
  uint32_t filled = 0, parity = ~0u;  // slots ever filled, parity of each one's last fill
  bool lost = wait_cycles <= 1;  // one cycle is over before the first look

  __device__ uint8_t* slot(uint32_t s, int row) const { return base + (s * ROWS + row) * room; }
  // Bytes of the words around a row.
  __device__ uint32_t words(const uint8_t* row) const { return (row_offset(row) + row_bytes + 15) & ~15u; }
  // One thread: the rows of one token into slot s (a null row is left out).
  __device__ void fill(uint32_t s, const uint8_t* const (&rows)[ROWS]) {
    uint32_t bytes = 0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) bytes += rows[r] ? words(rows[r]) : 0;
    mbar_arrive_expect_tx(&full[s], bytes);
    filled |= 1u << s;
    parity ^= 1u << s;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (rows[r]) bulk_load_1d(slot(s, r), rows[r] - row_offset(rows[r]), words(rows[r]), &full[s]);
  }
  __device__ void wait() {
    if (!lost) lost = !mbar_wait_bounded(&full[stage], phase, wait_cycles);
  }
  // The filling thread, last: its copies have landed before the block exits.
  __device__ void drain() const {
    for (uint32_t s = 0; s < stages; ++s)
      if (filled & (1u << s)) (void)mbar_wait_bounded(&full[s], (parity >> s) & 1u);
  }
  __device__ void next() {
    if (++stage == stages) stage = 0, phase ^= 1u;
  }
};

// The streamed forward form: dim a multiple of 8, at most NV vectors a thread.
template <typename T, typename W, int NV>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_stream_kernel(const Forward p, int64_t tokens, uint32_t stages) {
  extern __shared__ __align__(16) uint8_t ring_bytes[];
  __shared__ __align__(8) uint64_t full[kMaxRing];
  __shared__ SumSlots<1> slots[2][2];
  __shared__ uint32_t max_slots[2][32];
  const int n = blockDim.x, tid = threadIdx.x;
  for (int b = 0; b < 4; ++b) clear_slots(slots[b / 2][b % 2]);
  const uint32_t row_bytes = p.dim * sizeof(T);
  RowRing<2> ring{ring_bytes, full, row_bytes, row_bytes, stages, p.wait_cycles};
  if (tid == 0) {
    for (uint32_t s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  __syncthreads();
  wait_previous_launch();
  allow_next_launch();
  const T* xs = static_cast<const T*>(p.x);
  const T* ys = static_cast<const T*>(p.y);
  auto fill = [&](uint32_t s, int64_t t) {
    const uint8_t* rows[2] = {reinterpret_cast<const uint8_t*>(xs + t * p.ld_x),
                              reinterpret_cast<const uint8_t*>(ys + t * p.ld_y)};
    ring.fill(s, rows);
  };
  if (tid == 0)
    for (uint32_t s = 0; s < stages && blockIdx.x + static_cast<int64_t>(s) * gridDim.x < tokens; ++s)
      fill(s, blockIdx.x + static_cast<int64_t>(s) * gridDim.x);

  int buf = 0;
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x, buf ^= 1) {
    ring.wait();
    F2 y[NV][4], v[NV][4];
    Raw8<T> x[NV];
    auto take = [&](const T* xrow, const T* yrow) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = (j * n + tid) * 8;
        load8<true>(yrow, p.dim, j, n, tid, y[j]);
        x[j].load(xrow + i, i < p.dim);
      }
    };
    if (!ring.lost)  // two branches, so that these are shared-memory loads
      take(reinterpret_cast<const T*>(ring.slot(ring.stage, 0)), reinterpret_cast<const T*>(ring.slot(ring.stage, 1)));
    else
      take(xs + t * p.ld_x, ys + t * p.ld_y);
    release_stage_reads();
    // The reduction's barrier also tells the filling thread that the slot is
    // read, so it runs without a norm of y too.
    const float squares = row_squares(y, slots[buf][0]);
    if (n == 32) __syncwarp();
    const float f = p.post ? p.scale * rsqrtf(squares * p.inv_dim + p.eps) : p.scale;
    if (tid == 0 && !ring.lost && t + static_cast<int64_t>(stages) * gridDim.x < tokens)
      fill(ring.stage, t + static_cast<int64_t>(stages) * gridDim.x);
    ring.next();

    const W* gate = static_cast<const W*>(p.gate) + (p.gate ? t / p.rows_per_gate * p.ld_gate : 0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = x[j].pair(e);
      add_update<Access::Words, T, W>(p, gate, f, j, n, tid, y[j], v[j]);
      store8<true>(static_cast<T*>(p.x_out) + t * p.ld_x_out, p.dim, j, n, tid, v[j]);
    }
    if (!p.pre) continue;
    const float rho = rsqrtf(row_squares(v, slots[buf][1]) * p.inv_dim + p.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      normalize<Access::Words, W>(p, rho, j, n, tid, v[j]);
      if (p.h) store8<true>(static_cast<T*>(p.h) + t * p.ld_h, p.dim, j, n, tid, v[j]);
    }
    if (!p.q) continue;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) top = max(top, row_magnitude<Access::Words>(v[j], p.dim, j, n, tid));
    const RowScale rs = make_row_scale(block_max(top, max_slots[buf]));
    if (tid == 0) p.q_scale[t] = rs.scale;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_q8<true>(p.q + t * p.ld_q, p.dim, j, n, tid, v[j], rs.inv);
  }
  if (tid == 0) ring.drain();
}

struct Backward {
  int64_t ld_dxo, ld_dh, ld_x, ld_y, ld_gate, ld_dx, ld_dy, ld_dgate;
  const void *dxo, *dh, *x, *y, *post, *pre, *gate;
  void *dx, *dy, *dgate;
  float *part_post, *part_pre, *part_gate;  // per-block sums [grid][pitch], per-item gate sums [items][pitch]
  int64_t tokens, items, chunks, rows_per_item, rows_per_group, rows_per_gate;
  // The offsets are added to a weight; of an absent one, read as zeros, they are
  // the whole factor.
  float scale, eps, pre_offset, inv_dim;
  float post_offset;
  int dim, pitch;
  // Elements of x and y that are read: what takes no part counts as zeros, an
  // infinity in it would make a NaN of every product with 0 (x without a norm of
  // it, y without a norm of it or a gate's gradient). A branch around the loads
  // costs more (4000 x 8191 f32 197 us, 222).
  int x_dim, y_dim;
  bool per_token;  // one gate row per token: d_gate is written token by token
  bool dgate_f32;  // in 32 bits then too (W of 32 bits only)
  int64_t wait_cycles;
};

// What the two backward forms share, for one vector of a row.
template <Access A, typename T>
__device__ __forceinline__ void load_or(const T* row, float none, int dim, int j, int n, int tid, F2 (&v)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = f2(none);
  if (row) load_row<A>(row, dim, j, n, tid, v);
}
// a = scale * gate * (offset + post), pre = offset + pre_weight (0 without).
template <Access A, typename W>
__device__ __forceinline__ void make_factors(const Backward& p, const W* gate, int j, int n, int tid, F2 (&a)[4],
                                             F2 (&pre)[4]) {
  F2 w[4], g[4];
  load_or<A>(static_cast<const W*>(p.post), 0.0f, p.dim, j, n, tid, w);
  load_or<A>(p.gate ? gate : nullptr, 1.0f, p.dim, j, n, tid, g);
  load_or<A>(static_cast<const W*>(p.pre), -p.pre_offset, p.dim, j, n, tid, pre);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    a[e] = f2(p.scale) * g[e] * (w[e] + f2(p.post_offset));
    pre[e] = pre[e] + f2(p.pre_offset);
  }
}
// u dx summed or single -> the gate's gradient in place, post's share added.
template <Access A, typename W>
__device__ __forceinline__ void gate_gradient(const Backward& p, const W* gate, int j, int n, int tid, F2 (&udx)[4],
                                              F2 (&acc_post)[4]) {
  F2 w[4], g[4];
  load_or<A>(static_cast<const W*>(p.post), 0.0f, p.dim, j, n, tid, w);
  load_or<A>(p.gate ? gate : nullptr, 1.0f, p.dim, j, n, tid, g);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    acc_post[e] = fma(f2(p.scale) * g[e], udx[e], acc_post[e]);
    udx[e] = f2(p.scale) * (w[e] + f2(p.post_offset)) * udx[e];
  }
}
// A token's own gate gradient.
template <Access A, typename T, typename W>
__device__ __forceinline__ void store_token_gate(const Backward& p, int64_t t, int j, int n, int tid, const F2 (&v)[4]) {
  if constexpr (sizeof(T) < sizeof(W)) {
    if (p.dgate_f32) return store_row<A>(static_cast<float*>(p.dgate) + t * p.ld_dgate, p.dim, j, n, tid, v);
  }
  store_row<A>(static_cast<T*>(p.dgate) + t * p.ld_dgate, p.dim, j, n, tid, v);
}
// A row needs one reduction: with a = scale * gate * (offset + post),
// mean(v u) expands over dx = dxo + rho (t - mean(t n) n) into sums that do
// not depend on dx.
struct RowSums {
  F2 xx, tx, yy, yd, yt, yx;
  __device__ __forceinline__ void add(const F2 (&dxo)[4], const F2 (&dh)[4], const F2 (&x)[4], const F2 (&y)[4],
                                      const F2 (&a)[4], const F2 (&pre)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const F2 t = dh[e] * pre[e], ay = a[e] * y[e];
      xx = fma(x[e], x[e], xx);
      tx = fma(t, x[e], tx);
      yy = fma(y[e], y[e], yy);
      yd = fma(ay, dxo[e], yd);
      yt = fma(ay, t, yt);
      yx = fma(ay, x[e], yx);
    }
  }
};
// Rows far from 1 in magnitude: x and y meet their row factors as n = rho x and
// u = sigma y, and the means are of the gradients' size, so that no power of a
// row factor is formed; rho^3 or sigma^2 mean(v u) leave the 32-bit range for
// rows whose rms is past 1e13 or below 1e-13. Two products a pair of elements
// more than with powers (us: 16384 x 4096 bf16 143, 140 with them; 8192 x 8192
// 144 and 143.5; 4000 x 8191 171 and 168).
struct RowFactors {
  F2 rho, minus_tn, sigma, minus_vu;  // 1/rms(x), -mean(t n), 1/rms(y), -mean(v u)
};
__device__ __forceinline__ RowFactors row_factors(const Backward& p, const RowSums& sums, SumSlots<6>& slots) {
  float s[6] = {both(sums.xx), both(sums.tx), both(sums.yy), both(sums.yd), both(sums.yt), both(sums.yx)};
  block_sum(s, slots);
  const float rho = p.pre ? rsqrtf(s[0] * p.inv_dim + p.eps) : 0.0f;
  const float mtn = rho * s[1] * p.inv_dim;
  const float sigma = p.post ? rsqrtf(s[2] * p.inv_dim + p.eps) : 1.0f;
  const float mvu = p.post ? sigma * (s[3] + rho * (s[4] - mtn * (rho * s[5]))) * p.inv_dim : 0.0f;
  return RowFactors{f2(rho), f2(-mtn), f2(sigma), f2(-mvu)};
}
__device__ __forceinline__ void row_gradients(const RowFactors& r, const F2 (&dxo)[4], const F2 (&dh)[4],
                                              const F2 (&x)[4], const F2 (&y)[4], const F2 (&a)[4], const F2 (&pre)[4],
                                              F2 (&dx)[4], F2 (&dy)[4], F2 (&udx)[4], F2 (&acc_pre)[4], bool post) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const F2 n = r.rho * x[e], u = r.sigma * y[e];
    dx[e] = fma(r.rho, fma(r.minus_tn, n, dh[e] * pre[e]), dxo[e]);
    acc_pre[e] = fma(dh[e], n, acc_pre[e]);
    dy[e] = a[e] * dx[e];
    if (post) dy[e] = r.sigma * fma(r.minus_vu, u, dy[e]);  // without a norm of y, no value of y (0 * infinity)
    udx[e] = u * dx[e];
  }
}

constexpr int kNarrow = 4096;  // widest row of the direct backward form's blocks with a vector a thread

// A block walks items (runs of tokens that share a gate row) and keeps the
// sums over tokens in registers: for dgate and dpost A = sum of u * dx over an
// item (both are multiples of it by per-channel factors), for dpre its own. With
// NV = 4 (past 8192 columns) the registers of so many threads do not hold a
// vector's values: 0.5 to 1.1 KB a thread spill, and the row is read twice (us:
// 4096 x 16384 bf16 610, where HBM needs 125; 1000 x 16383 760).
template <typename T, typename W, Access A, int NV>
__global__ void __launch_bounds__(NV == 1 ? kNarrow / 8 : kMaxThreads) residual_norm_backward_kernel(const Backward p) {
  __shared__ SumSlots<6> slots[2];
  const int n = blockDim.x, tid = threadIdx.x;
  clear_slots(slots[0]);
  clear_slots(slots[1]);
  __syncthreads();
  wait_previous_launch();
  allow_next_launch();
  F2 acc_pre[NV][4] = {}, acc_post[NV][4] = {};
  int buf = 0;
  for (int64_t item = blockIdx.x; item < p.items; item += gridDim.x) {
    const int64_t group = item / p.chunks, first = group * p.rows_per_group + (item % p.chunks) * p.rows_per_item;
    const int64_t last = min(first + p.rows_per_item, (group + 1) * p.rows_per_group);
    F2 acc[NV][4] = {};
    for (int64_t t = first; t < last; ++t, buf ^= 1) {
      const T* dxo = p.dxo ? static_cast<const T*>(p.dxo) + t * p.ld_dxo : nullptr;
      const T* dh = p.dh ? static_cast<const T*>(p.dh) + t * p.ld_dh : nullptr;
      const T* x = static_cast<const T*>(p.x) + t * p.ld_x;
      const T* y = static_cast<const T*>(p.y) + t * p.ld_y;
      const W* gate = p.gate ? static_cast<const W*>(p.gate) + t / p.rows_per_gate * p.ld_gate : nullptr;
      struct Vec {
        F2 dxo[4], dh[4], x[4], y[4], a[4], pre[4];
      };
      auto load = [&](int j, Vec& v) {
        load_row<A>(x, p.x_dim, j, n, tid, v.x);
        load_row<A>(y, p.y_dim, j, n, tid, v.y);
        load_or<A>(dxo, 0.0f, p.dim, j, n, tid, v.dxo);
        load_or<A>(dh, 0.0f, p.dim, j, n, tid, v.dh);
        make_factors<A, W>(p, gate, j, n, tid, v.a, v.pre);
      };
      Vec v;
      RowSums sums{};
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        load(j, v);
        sums.add(v.dxo, v.dh, v.x, v.y, v.a, v.pre);
      }
      const RowFactors r = row_factors(p, sums, slots[buf]);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (NV > 1) load(j, v);
        F2 dx[4], dy[4], udx[4];
        row_gradients(r, v.dxo, v.dh, v.x, v.y, v.a, v.pre, dx, dy, udx, acc_pre[j], p.post);
        store_row<A>(static_cast<T*>(p.dx) + t * p.ld_dx, p.dim, j, n, tid, dx);
        store_row<A>(static_cast<T*>(p.dy) + t * p.ld_dy, p.dim, j, n, tid, dy);
        if (p.per_token) {
          gate_gradient<A, W>(p, gate, j, n, tid, udx, acc_post[j]);
          if (p.dgate) store_token_gate<A, T, W>(p, t, j, n, tid, udx);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] = acc[j][e] + udx[e];
        }
      }
    }
    if (!p.per_token) {
      const W* gate = static_cast<const W*>(p.gate) + (p.gate ? first / p.rows_per_gate * p.ld_gate : 0);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        gate_gradient<A, W>(p, gate, j, n, tid, acc[j], acc_post[j]);
        if (p.part_gate)
          store_partial<A>(p.part_gate + item * p.pitch, p.dim, j, n, tid, acc[j]);
        else if (p.dgate)
          store_row<A>(static_cast<float*>(p.dgate) + group * p.ld_dgate, p.dim, j, n, tid, acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (p.part_post) store_partial<A>(p.part_post + static_cast<int64_t>(blockIdx.x) * p.pitch, p.dim, j, n, tid, acc_post[j]);
    if (p.part_pre) store_partial<A>(p.part_pre + static_cast<int64_t>(blockIdx.x) * p.pitch, p.dim, j, n, tid, acc_pre[j]);
  }
}

// The streamed backward form. Per element it does some 30 operations for 12
// bytes, half of what an SM can issue at its share of HBM, so the token's words
// are read once and the per-channel factors are made once while the gate row
// lasts, in shared memory (a thread reads back its own, conflict-free); the
// registers hold the row and two sums a channel. NV vectors a thread keep what
// a row costs besides its elements (one reduction of six sums) small.
// With a gate row per token (PER_TOKEN) the gate's words are copied with the
// token's (GATE_COPIED) or brought to L2 with them, and the factors kept are
// those of the weights alone.
template <typename T, typename W, Access A, int NV, bool PER_TOKEN, bool GATE_COPIED>
__global__ void __launch_bounds__(512) residual_norm_backward_stream_kernel(const Backward p, uint32_t stages) {
  extern __shared__ __align__(16) uint8_t ring_bytes[];
  __shared__ __align__(8) uint64_t full[kMaxRing];
  __shared__ SumSlots<6> slots[2];
  const int n = blockDim.x, tid = threadIdx.x;
  clear_slots(slots[0]);
  clear_slots(slots[1]);
  constexpr int ROWS = GATE_COPIED ? 5 : 4;
  RowRing<ROWS> ring{ring_bytes, full, static_cast<uint32_t>(p.dim * sizeof(T)),
                     row_room(A == Access::Words, p.dim, sizeof(T)), stages, p.wait_cycles};
  float4* factors = reinterpret_cast<float4*>(ring_bytes + stages * ROWS * ring.room);  // [NV][4][n]: a, a, pre, pre
  if (tid == 0) {
    for (uint32_t s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  __syncthreads();
  wait_previous_launch();
  allow_next_launch();

  // This block's tokens in order: runs of rows_per_item from its items.
  struct Cursor {
    int item, t, last;
  };
  const int items = static_cast<int>(p.items), chunks = static_cast<int>(p.chunks);
  auto enter = [&](Cursor& c) {
    if (c.item >= items) return;
    const int group = c.item / chunks;
    c.t = static_cast<int>(group * p.rows_per_group + (c.item - group * chunks) * p.rows_per_item);
    c.last = static_cast<int>(min(c.t + p.rows_per_item, (group + 1) * p.rows_per_group));
  };
  auto advance = [&](Cursor& c) {
    if (++c.t == c.last) {
      c.item += gridDim.x;
      enter(c);
    }
  };
  const T* dxo_base = static_cast<const T*>(p.dxo);
  const T* dh_base = static_cast<const T*>(p.dh);
  const T* x_base = static_cast<const T*>(p.x);
  const T* y_base = static_cast<const T*>(p.y);
  const T* bases[4] = {dxo_base, dh_base, x_base, y_base};
  const int64_t lds[4] = {p.ld_dxo, p.ld_dh, p.ld_x, p.ld_y};
  auto fill = [&](uint32_t s, int64_t t) {
    const bool copy = copied<A>(t, p.tokens);
    const uint8_t* rows[ROWS];
#pragma unroll
    for (int r = 0; r < 4; ++r) rows[r] = reinterpret_cast<const uint8_t*>(bases[r] && copy ? bases[r] + t * lds[r] : nullptr);
    if (GATE_COPIED)
      rows[ROWS - 1] = reinterpret_cast<const uint8_t*>(copy ? static_cast<const W*>(p.gate) + t * p.ld_gate : nullptr);
    if (PER_TOKEN && copy && !GATE_COPIED) {
      const W* gate = static_cast<const W*>(p.gate) + t * p.ld_gate;
      prefetch_l2(reinterpret_cast<const uint8_t*>(gate) - row_offset(gate),
                  (row_offset(gate) + p.dim * static_cast<uint32_t>(sizeof(W)) + 15) & ~15u);
    }
    ring.fill(s, rows);
  };
  Cursor ahead{static_cast<int>(blockIdx.x), 0, 0};
  if (tid == 0) {
    enter(ahead);
    for (uint32_t s = 0; s < stages && ahead.item < items; ++s, advance(ahead)) fill(s, ahead.t);
  }

  // The factors of this thread's channels in shared memory, read back by it alone.
  auto keep_factors = [&](int t) {
    const W* gate = PER_TOKEN || !p.gate ? nullptr : static_cast<const W*>(p.gate) + t / p.rows_per_gate * p.ld_gate;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      F2 a[4], pre[4];
      make_factors<A, W>(p, gate, j, n, tid, a, pre);
      float4* f = factors + j * 4 * n + tid;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f[h * n] = make_float4(a[2 * h].v.x, a[2 * h].v.y, a[2 * h + 1].v.x, a[2 * h + 1].v.y);
        f[(2 + h) * n] = make_float4(pre[2 * h].v.x, pre[2 * h].v.y, pre[2 * h + 1].v.x, pre[2 * h + 1].v.y);
      }
    }
  };
  auto get_factors = [&](int j, F2 (&a)[4], F2 (&pre)[4]) {
    const float4* f = factors + j * 4 * n + tid;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 fa = f[h * n], fp = f[(2 + h) * n];
      a[2 * h] = f2(fa.x, fa.y), a[2 * h + 1] = f2(fa.z, fa.w);
      pre[2 * h] = f2(fp.x, fp.y), pre[2 * h + 1] = f2(fp.z, fp.w);
    }
  };
  F2 acc_pre[NV][4] = {}, acc[NV][4] = {};
  int buf = 0;
  Cursor now{static_cast<int>(blockIdx.x), 0, 0};
  enter(now);
  bool fresh = true;  // the gate row changed
  while (now.item < items) {
    const int item = now.item;
    const int64_t t = now.t;
    if (fresh) keep_factors(now.t);
    Raw8<W> gate_row[PER_TOKEN ? NV : 1];
    auto take_gate = [&](const W* row) {
#pragma unroll
      for (int j = 0; j < NV; ++j) gate_row[j] = load_raw<A>(row, p.dim, j, n, tid);
    };
    const W* token_gate = PER_TOKEN ? static_cast<const W*>(p.gate) + t * p.ld_gate : nullptr;
    if (PER_TOKEN && !GATE_COPIED) take_gate(token_gate);
    ring.wait();
    Raw8<T> dxo[NV], dh[NV], x[NV], y[NV];
    auto take = [&](auto row) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        dxo[j] = dh[j] = Raw8<T>{};
        if (dxo_base) dxo[j] = load_raw<A>(row(0), p.dim, j, n, tid);
        if (dh_base) dh[j] = load_raw<A>(row(1), p.dim, j, n, tid);
        x[j] = load_raw<A>(row(2), p.x_dim, j, n, tid);
        y[j] = load_raw<A>(row(3), p.y_dim, j, n, tid);
      }
    };
    // Two branches, so that these are shared-memory loads.
    if (!ring.lost && copied<A>(t, p.tokens)) {
      take([&](int r) { return reinterpret_cast<const T*>(ring.slot(ring.stage, r) + row_offset(bases[r] + t * lds[r])); });
      if constexpr (GATE_COPIED) take_gate(reinterpret_cast<const W*>(ring.slot(ring.stage, 4) + row_offset(token_gate)));
    } else {
      take([&](int r) { return bases[r] + t * lds[r]; });
      if (GATE_COPIED) take_gate(token_gate);
    }
    release_stage_reads();
    RowSums sums{};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      F2 fdxo[4], fdh[4], fx[4], fy[4], a[4], pre[4];
      get_factors(j, a, pre);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        fdxo[e] = dxo[j].pair(e), fdh[e] = dh[j].pair(e), fx[e] = x[j].pair(e), fy[e] = y[j].pair(e);
      if (PER_TOKEN)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = a[e] * gate_row[j].pair(e);
      sums.add(fdxo, fdh, fx, fy, a, pre);
    }
    const RowFactors r = row_factors(p, sums, slots[buf]);
    buf ^= 1;
    if (n == 32) __syncwarp();
    if (tid == 0 && !ring.lost && ahead.item < items) {
      fill(ring.stage, ahead.t);
      advance(ahead);
    }
    ring.next();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      F2 dx[4], dy[4], udx[4];
      {
        F2 fdxo[4], fdh[4], fx[4], fy[4], a[4], pre[4];
        get_factors(j, a, pre);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          fdxo[e] = dxo[j].pair(e), fdh[e] = dh[j].pair(e), fx[e] = x[j].pair(e), fy[e] = y[j].pair(e);
        if (PER_TOKEN)
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = a[e] * gate_row[j].pair(e);
        row_gradients(r, fdxo, fdh, fx, fy, a, pre, dx, dy, udx, acc_pre[j], p.post);
      }
      store_row<A>(static_cast<T*>(p.dx) + t * p.ld_dx, p.dim, j, n, tid, dx);
      store_row<A>(static_cast<T*>(p.dy) + t * p.ld_dy, p.dim, j, n, tid, dy);
      if (PER_TOKEN) {
        F2 base[4], pre[4];  // scale * (offset + post)
        get_factors(j, base, pre);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[j][e] = fma(f2(p.scale) * gate_row[j].pair(e), udx[e], acc[j][e]);
          udx[e] = base[e] * udx[e];
        }
        if (p.dgate) store_token_gate<A, T, W>(p, t, j, n, tid, udx);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = acc[j][e] + udx[e];
      }
    }
    advance(now);
    const bool ended = now.item != item;
    fresh = !PER_TOKEN && ended;
    if (PER_TOKEN || !ended) continue;
    // The item's sums: its gate row's gradient, and its share of post's, which
    // the block adds up over its items in its own row of part_post.
    const W* gate = static_cast<const W*>(p.gate) + (p.gate ? t / p.rows_per_gate * p.ld_gate : 0);
    float* dp = p.part_post ? p.part_post + static_cast<int64_t>(blockIdx.x) * p.pitch : nullptr;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      F2 post[4] = {};
      if (dp && item != static_cast<int>(blockIdx.x)) load8<A != Access::Elements>(dp, p.dim, j, n, tid, post);
      gate_gradient<A, W>(p, gate, j, n, tid, acc[j], post);
      if (dp) store_partial<A>(dp, p.dim, j, n, tid, post);
      if (p.part_gate)
        store_partial<A>(p.part_gate + static_cast<int64_t>(item) * p.pitch, p.dim, j, n, tid, acc[j]);
      else if (p.dgate)
        store_row<A>(static_cast<float*>(p.dgate) + item / chunks * p.ld_dgate, p.dim, j, n, tid, acc[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = f2(0.0f);
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (p.part_post && PER_TOKEN)
      store_partial<A>(p.part_post + static_cast<int64_t>(blockIdx.x) * p.pitch, p.dim, j, n, tid, acc[j]);
    if (p.part_pre) store_partial<A>(p.part_pre + static_cast<int64_t>(blockIdx.x) * p.pitch, p.dim, j, n, tid, acc_pre[j]);
  }
  if (tid == 0) ring.drain();
}

// out[g][c] = sum over the group's `count` consecutive rows of part. A block
// sums 32 columns, four a thread, over the rows that THREADS / 8 row lanes take
// in turn, always in the same order (rows are padded to whole words); four rows
// a lane are on their way at once. blockIdx.y picks the sum: the first two have
// one group, the blocks after them walk the third's.
struct Sums {
  const float* part[3];
  float* out[3];
  int64_t count[3], groups, ld_out;
  int dim, pitch;
};
template <int THREADS>
__global__ void __launch_bounds__(THREADS) sum_rows_kernel(const Sums p) {
  __shared__ float4 s[THREADS / 32][8];
  constexpr int ROWS = THREADS / 8;
  wait_previous_launch();
  allow_next_launch();
  const bool third = blockIdx.y >= 2;
  float* out = third ? p.out[2] : blockIdx.y ? p.out[1] : p.out[0];
  if (!out) return;
  const float* base = third ? p.part[2] : blockIdx.y ? p.part[1] : p.part[0];
  const int count = static_cast<int>(third ? p.count[2] : blockIdx.y ? p.count[1] : p.count[0]);
  const int64_t groups = third ? p.groups : 1, step = third ? gridDim.y - 2 : 1;
  const int c = blockIdx.x * 32 + threadIdx.x % 8 * 4, lane = threadIdx.x / 8;
  for (int64_t g = third ? blockIdx.y - 2 : 0; g < groups; g += step) {
    const float* part = base + g * count * p.pitch + c;
    float4 v = make_float4(0, 0, 0, 0);
    auto add = [&](const float4& a) { v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w; };
    if (c < p.dim)
      for (int r = lane; r < count; r += 4 * ROWS) {
        float4 a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          a[i] = r + i * ROWS < count ? *reinterpret_cast<const float4*>(part + static_cast<int64_t>(r + i * ROWS) * p.pitch)
                                      : make_float4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) add(a[i]);
      }
#pragma unroll
    for (int o = 8; o < 32; o <<= 1)
      add(make_float4(__shfl_xor_sync(0xFFFFFFFFu, v.x, o), __shfl_xor_sync(0xFFFFFFFFu, v.y, o),
                      __shfl_xor_sync(0xFFFFFFFFu, v.z, o), __shfl_xor_sync(0xFFFFFFFFu, v.w, o)));
    if (threadIdx.x % 32 < 8) s[threadIdx.x / 32][threadIdx.x % 8] = v;
    __syncthreads();
    if (threadIdx.x < 32 && blockIdx.x * 32 + threadIdx.x < p.dim) {
      float all = 0.0f;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) all += reinterpret_cast<const float*>(s[w])[threadIdx.x];
      out[g * p.ld_out + blockIdx.x * 32 + threadIdx.x] = all;
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

// Calls f(T, W).
template <typename F>
cudaError_t dispatch_types(uint32_t type, uint32_t weight_type, F&& f) {
  if (type == RNS8_CUDA_TYPE_F32) return f(float{}, float{});
  if (type == RNS8_CUDA_TYPE_BF16)
    return weight_type == RNS8_CUDA_TYPE_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
  return weight_type == RNS8_CUDA_TYPE_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
}

// A streamed kernel's launch: vectors and threads a block, blocks an SM (by
// the registers those take), slots of the ring.
struct Stream {
  int nv;
  unsigned threads, per_sm, stages;
  size_t smem;
};
constexpr size_t kSmemOfSm = 220 * 1024;  // for the dynamic shared memory of an SM's blocks
// The forward ring stays small: HBM needs some 45 KB of an SM in flight, and
// the rest of the SM's memory caches the weights, which every token reads
// again (8192 x 8192 bf16: 97 us; 111 us with a ring of three rows a block).
constexpr size_t kForwardSmemOfSm = 64 * 1024;

Stream forward_stream(int dim, size_t elem) {
  const int vecs = dim / 8;
  Stream s{};
  s.nv = vecs <= 32 ? 1 : 2;
  s.threads = block_threads(dim, s.nv);
  s.per_sm = std::max(1u, std::min(16u, 1024 / s.threads));
  const size_t slot = 2 * static_cast<size_t>(dim) * elem;
  s.stages = static_cast<unsigned>(std::min<size_t>(kMaxRing, std::max<size_t>(1, kForwardSmemOfSm / s.per_sm / slot)));
  s.smem = s.stages * slot;
  return s;
}

// The backward pass. Its grid depends on the sizes alone, so that the scratch
// for the blocks' sums does too.
Stream backward_stream(int dim, size_t elem, bool aligned, int rows) {
  const int vecs = (dim + 7) / 8;
  Stream s{};
  s.nv = vecs <= 64 ? 1 : 2;
  s.threads = block_threads(dim, s.nv);
  s.per_sm = std::max(1u, std::min(8u, 512 / s.threads));
  const size_t slot = rows * static_cast<size_t>(row_room(aligned, dim, static_cast<uint32_t>(elem)));
  const size_t factors = 64 * static_cast<size_t>(s.nv) * s.threads;
  const size_t room = kSmemOfSm / s.per_sm;
  s.stages = static_cast<unsigned>(room > factors ? std::min<size_t>(kMaxRing, (room - factors) / slot) : 0);
  s.smem = s.stages * slot + factors;
  return s;
}
int padded(int64_t dim) { return static_cast<int>((dim + 7) / 8 * 8); }

// How the backward pass splits its tokens: items of one gate row each, at
// most `chunks` items per gate row, walked by `grid` blocks.
struct Split {
  int64_t groups, rows_per_group, chunks, rows_per_item, items;
  int64_t grid;
  bool per_token;
};
Split split_tokens(const rns8_cuda_residual_norm_backward_desc& d, int sm_count) {
  Split s;
  const Stream st = backward_stream(static_cast<int>(d.dim), type_size(d.type), true, 4);
  const int64_t target = static_cast<int64_t>(st.per_sm) * sm_count;
  s.per_token = d.gate && d.groups == d.tokens;
  s.groups = (s.per_token || !d.gate) ? 1 : d.groups;
  s.rows_per_group = d.tokens / s.groups;
  // No more items than blocks where the groups allow it: a second item would
  // double a block's time.
  s.chunks = std::min(s.rows_per_group, std::max<int64_t>(1, target / s.groups));
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

cudaError_t residual_norm(const rns8_cuda_residual_norm_desc& d, int sm_count, cudaStream_t stream) {
  Forward p{};
  p.rows_per_gate = d.gate ? d.tokens / d.groups : 1;
  p.ld_x = d.ld_x, p.ld_y = d.ld_y, p.ld_gate = d.ld_gate, p.ld_x_out = d.ld_x_out, p.ld_h = d.ld_h, p.ld_q = d.ld_q;
  p.x = d.x, p.y = d.y, p.post = d.post_weight, p.pre = d.pre_weight, p.gate = d.gate;
  p.x_out = d.x_out, p.h = d.h, p.q = d.q, p.q_scale = d.q_scale;
  p.scale = d.scale, p.eps = d.eps, p.offset = d.weight_offset, p.dim = static_cast<int>(d.dim);
  p.inv_dim = 1.0f / static_cast<float>(p.dim);
  p.wait_cycles = quant_wait_cycles();
  p.q_words = reinterpret_cast<uintptr_t>(d.q) % 8 == 0 && d.ld_q % 8 == 0;
  const size_t e = type_size(d.type), w = type_size(d.weight_type);
  const bool aligned = d.dim % 8 == 0 && aligned_rows(d.x, d.ld_x, e) && aligned_rows(d.y, d.ld_y, e) &&
                       aligned_rows(d.post_weight, 0, w) && aligned_rows(d.pre_weight, 0, w) &&
                       aligned_rows(d.gate, d.ld_gate, w) && aligned_rows(d.x_out, d.ld_x_out, e) &&
                       aligned_rows(d.h, d.ld_h, e) &&
                       (!d.q || p.q_words);
  // Below some four tokens an SM each block has one or two rows and nothing to
  // run ahead for: the direct form's shorter start wins.
  if (aligned && p.dim <= 16384 && d.tokens >= 4 * static_cast<int64_t>(sm_count)) {
    const Stream s = forward_stream(p.dim, e);
    auto launch_stream = [&](auto t, auto wt, auto nv) {
      auto kernel = residual_norm_stream_kernel<decltype(t), decltype(wt), decltype(nv)::value>;
      static std::atomic<uint64_t> configured{0};
      const cudaError_t err = raise_smem_limit_once(kernel, static_cast<int>(kSmemOfSm), configured);
      if (err != cudaSuccess) return err;
      const int64_t grid = std::min<int64_t>(d.tokens, static_cast<int64_t>(s.per_sm) * sm_count);
      return launch_chained(kernel, dim3(static_cast<unsigned>(grid)), s.threads, s.smem, 1, stream, p, d.tokens,
                            s.stages);
    };
    return dispatch_types(d.type, d.weight_type, [&](auto t, auto wt) {
      return s.nv == 1 ? launch_stream(t, wt, std::integral_constant<int, 1>{})
                       : launch_stream(t, wt, std::integral_constant<int, 2>{});
    });
  }
  const int vectors = row_vectors(d.tokens, (p.dim + 7) / 8);
  return dispatch(d.type, d.weight_type, aligned, vectors, [&](auto t, auto wt, auto al, auto nv) {
    constexpr int NV = decltype(nv)::value;
    constexpr Access A = decltype(al)::value                      ? Access::Words
                         : NV == 1 && sizeof(decltype(t)) == 4 ? Access::Elements
                                                               : Access::Shifted;
    return launch_chained(residual_norm_kernel<decltype(t), decltype(wt), A, NV>,
                          dim3(static_cast<unsigned>(d.tokens)), block_threads(p.dim, NV), 0, 1, stream, p);
  });
}

uint64_t residual_norm_backward_scratch_bytes(const rns8_cuda_residual_norm_backward_desc& d, int sm_count) {
  const Split s = split_tokens(d, sm_count);
  uint64_t rows = 0;
  if (d.d_post) rows += s.grid;
  if (d.d_pre) rows += s.grid;
  if (gate_partials(d, s)) rows += s.items;
  return rows * static_cast<uint64_t>(padded(d.dim)) * sizeof(float) + (rows ? 16 : 0);
}

cudaError_t residual_norm_backward(const rns8_cuda_residual_norm_backward_desc& d, int sm_count, cudaStream_t stream) {
  const Split s = split_tokens(d, sm_count);
  Backward p{};
  p.ld_dxo = d.ld_d_x_out, p.ld_dh = d.ld_d_h, p.ld_x = d.ld_x_out, p.ld_y = d.ld_y, p.ld_gate = d.ld_gate;
  p.ld_dx = d.ld_d_x, p.ld_dy = d.ld_d_y, p.ld_dgate = d.ld_d_gate;
  p.dxo = d.d_x_out, p.dh = d.pre_weight ? d.d_h : nullptr, p.x = d.x_out, p.y = d.y;
  p.post = d.post_weight, p.pre = d.pre_weight, p.gate = d.gate;
  p.dx = d.d_x, p.dy = d.d_y, p.dgate = d.gate ? d.d_gate : nullptr;
  p.tokens = d.tokens, p.pitch = padded(d.dim);
  p.items = s.items, p.chunks = s.chunks, p.rows_per_item = s.rows_per_item, p.rows_per_group = s.rows_per_group;
  p.rows_per_gate = d.gate ? d.tokens / d.groups : 1;
  p.per_token = s.per_token;
  p.dgate_f32 = d.flags & RNS8_CUDA_NORM_D_GATE_F32;
  p.scale = d.scale, p.eps = d.eps, p.dim = static_cast<int>(d.dim);
  p.inv_dim = 1.0f / static_cast<float>(p.dim);
  p.post_offset = d.post_weight ? d.weight_offset : 1.0f;
  p.pre_offset = d.pre_weight ? d.weight_offset : 0.0f;
  p.wait_cycles = quant_wait_cycles();
  p.x_dim = d.pre_weight ? p.dim : 0;
  p.y_dim = d.post_weight || d.d_gate ? p.dim : 0;

  float* next = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(d.scratch) + 15) & ~uintptr_t(15));
  auto take = [&](int64_t rows) {
    float* at = next;
    next += rows * p.pitch;
    return at;
  };
  Sums sums{};
  sums.dim = p.dim, sums.pitch = p.pitch;
  if (d.d_post) {
    p.part_post = take(s.grid);
    sums.part[0] = p.part_post, sums.out[0] = d.d_post, sums.count[0] = s.grid;
  }
  if (d.d_pre) {
    p.part_pre = take(s.grid);
    sums.part[1] = p.part_pre, sums.out[1] = d.d_pre, sums.count[1] = s.grid;
  }
  if (gate_partials(d, s)) {
    p.part_gate = take(s.items);
    sums.part[2] = p.part_gate, sums.out[2] = static_cast<float*>(d.d_gate);
    sums.count[2] = s.chunks, sums.groups = s.groups, sums.ld_out = d.ld_d_gate;
  }

  const size_t e = type_size(d.type), w = type_size(d.weight_type);
  const bool aligned = d.dim % 8 == 0 && aligned_rows(d.d_x_out, d.ld_d_x_out, e) && aligned_rows(d.d_h, d.ld_d_h, e) &&
                       aligned_rows(d.x_out, d.ld_x_out, e) && aligned_rows(d.y, d.ld_y, e) &&
                       aligned_rows(d.post_weight, 0, w) && aligned_rows(d.pre_weight, 0, w) &&
                       aligned_rows(d.gate, d.ld_gate, w) && aligned_rows(d.d_x, d.ld_d_x, e) &&
                       aligned_rows(d.d_y, d.ld_d_y, e) &&
                       aligned_rows(d.d_gate, d.ld_d_gate, s.per_token && !p.dgate_f32 ? e : sizeof(float));
  // Per-token gate rows go through the ring too where two slots an SM remain (us:
  // 16384 x 4096 bf16 221, read beside it 282; 2000 x 8192, one slot, 80 and 70).
  Stream st = backward_stream(p.dim, e, aligned, 5);
  const bool gate_copied = aligned && s.per_token && e == w && st.stages * st.per_sm >= 2;
  if (!gate_copied) st = backward_stream(p.dim, e, aligned, 4);
  // A block with one row gains nothing from the ring and waits for its copies,
  // unless direct blocks, one an SM past 2048 columns, would run in turns (us,
  // direct and streamed, a gate row a token: 250 x 2048 f16 7.0 and 8.5; bf16 590 x
  // 1024 8.4 and 10.1, 148 x 4096 7.4 and 10.0, but 200 x 4096 11.5 and 10.7, 440 x
  // 2056 13.8 and 10.9). In turns too, floats on 16-byte boundaries (290 x 4096 16.9
  // and 18.8) and 16-bit rows off them (290 x 4095 17.4 and 19.7) go direct, floats
  // off them do not (440 x 2559 24.6 and 17.4). Where rows start anywhere the words
  // around them must lie within the matrix.
  const bool one_row = d.tokens <= static_cast<int64_t>(st.per_sm) * sm_count;
  const bool in_turns = p.dim > 2048 && d.tokens > sm_count && aligned == (e == 2);
  const bool streamed = p.dim <= 8192 && (aligned || p.dim >= 8) && !(one_row && !in_turns && p.dim <= kNarrow);
  const int vectors = streamed ? st.nv : p.dim <= kNarrow ? 1 : 4;
  const cudaError_t launched = dispatch(d.type, d.weight_type, aligned, vectors, [&](auto t, auto wt, auto al, auto nv) {
    using T = decltype(t);
    using W = decltype(wt);
    constexpr int NV = decltype(nv)::value;
    if (!streamed)
      return launch_chained(residual_norm_backward_kernel<T, W, al ? Access::Words : Access::Shifted, NV == 2 ? 1 : NV>,
                            dim3(static_cast<unsigned>(s.grid)), block_threads(p.dim, NV), 0, 1, stream, p);
    auto go = [&](auto per_token, auto gate_copied) {
      auto kernel = residual_norm_backward_stream_kernel<T, W, al ? Access::Words : Access::Elements, std::min(NV, 2),
                                                         decltype(per_token)::value, decltype(gate_copied)::value>;
      static std::atomic<uint64_t> configured{0};
      const cudaError_t bad = raise_smem_limit_once(kernel, static_cast<int>(kSmemOfSm), configured);
      if (bad != cudaSuccess) return bad;
      return launch_chained(kernel, dim3(static_cast<unsigned>(s.grid)), st.threads, st.smem, 1, stream, p, st.stages);
    };
    if constexpr (al && sizeof(T) == sizeof(W))
      if (gate_copied) return go(std::true_type{}, std::true_type{});
    return s.per_token ? go(std::true_type{}, std::false_type{}) : go(std::false_type{}, std::false_type{});
  });
  if (launched != cudaSuccess) return launched;
  cudaError_t err = cudaSuccess;
  if (sums.out[0] || sums.out[1] || sums.out[2]) {
    const unsigned walkers = sums.out[2] ? static_cast<unsigned>(std::min<int64_t>(s.groups, 1024)) : 0;
    const dim3 grid((p.dim + 31) / 32, 2 + walkers);
    // Few columns leave SMs idle unless blocks are wide, many groups do not (us,
    // pass with its sums, 512 and 256 threads: 2000 x 1024 bf16 16.6 and 24.1,
    // with 10 gate rows 2000 x 2048 22.5 and 25.0, 2000 x 8192 58.7 and 52.3).
    if (grid.x * grid.y <= 8u * sm_count)
      err = launch_chained(sum_rows_kernel<512>, grid, 512, 0, 1, stream, sums);
    else
      err = launch_chained(sum_rows_kernel<256>, grid, 256, 0, 1, stream, sums);
  }
  return err;
}

}  // namespace rns8cuda
