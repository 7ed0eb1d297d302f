/* 8-bit operators of large language models on the sm_100a backend: the int8
 * matrix product with a scale for each token and each output channel, the
 * quantisation of activations that feeds it, and the norms around a block
 * fused with its gate and residual update (forward, forward to int8 tokens,
 * backward).
 *
 * Like the rest of the device-pointer seam (rns8_cuda.h) every call takes
 * device pointers and a CUDA stream, only enqueues work, allocates nothing and
 * leaves the caller's current device as it found it. The arguments travel in
 * descriptors that begin with {uint64_t struct_size; uint32_t abi_version},
 * checked as in rns8.h. Scratch belongs to the call until its work on the
 * stream has run; its contents need no preparation.
 *
 * Matrices are row-major with a leading dimension counted in elements
 * (ld >= columns); no base pointer or leading dimension has an alignment rule
 * beyond the element's own size, but rows that start on 16-byte boundaries run
 * faster.
 *
 * Return value: RNS8_SUCCESS when the work was enqueued (also when there are
 * no rows: nothing is launched), RNS8_INVALID_ARGUMENT for malformed
 * arguments, RNS8_ACCUMULATION_OVERFLOW_RISK for a K beyond the exact range of
 * a 32-bit sum, RNS8_WORKSPACE_TOO_SMALL for too little scratch,
 * RNS8_BACKEND_FAILURE for a CUDA error. Outputs are untouched unless the
 * call returns RNS8_SUCCESS. */
#ifndef RNS8_RNS8_QUANT_H
#define RNS8_RNS8_QUANT_H

#include <stdint.h>

#include "rns8/abi.h"
#include "rns8/status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define RNS8_CUDA_TYPE_BF16 0u
#define RNS8_CUDA_TYPE_F16 1u
#define RNS8_CUDA_TYPE_F32 2u
#define RNS8_CUDA_TYPE_I8 3u

/* Symmetric quantisation of each row: with a = max |x| over the row,
 *   scale = a / 127,  q = round-half-to-even(x * (127 / a)),
 * every operation in 32-bit floats. A row whose scale would be subnormal
 * (a < 127 * 2^-126, an all-zero row among them) gets scale 0 and zeros. A row
 * with an infinity or a NaN gets that as its scale and zeros, so every product
 * with it is NaN. Bytes of q past `cols` are not written. */
typedef struct rns8_cuda_quantize_desc {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t flags; /* must be zero */
  int32_t device_id;
  uint32_t x_type; /* BF16, F16 or F32 */
  int64_t rows, cols, ld_x, ld_q;
  const void* x;
  int8_t* q;
  float* scale; /* [rows] */
  void* stream;
} rns8_cuda_quantize_desc;
RNS8_API rns8_status rns8_cuda_quantize_rows_device(const rns8_cuda_quantize_desc* desc);

/* Linear layer on 8-bit integers:
 *   acc[i][j] = sum over k of q[i][k] * w[j][k]          (exact, 32-bit)
 *   y[i][j]   = acc[i][j] * a_scale[i] * w_scale[j] + bias[j]
 * out = y rounded once to out_type. With RNS8_CUDA_LINEAR_GATED w holds 2n
 * rows, the first n the gate's: out = silu(y[i][j]) * y[i][n + j]. With out_type
 * I8 the result comes as int8 rows with their scales in out_scale, quantised as
 * above from its 32-bit values: the tokens of a next product, whose error then
 * holds no rounding to a 16-bit type in between.
 * a is either int8 rows with their scales (a_type I8) or floating rows that
 * the call quantises as rns8_cuda_quantize_rows_device does (a_scale NULL).
 * w is n (2n) rows of k int8, as a checkpoint keeps a layer's output channels.
 * k <= 131071: beyond that 32 bits may not hold the sum
 * (RNS8_ACCUMULATION_OVERFLOW_RISK). status receives 0x100 (ORed) if a bounded
 * device wait ran out; outputs are then unspecified. */
#define RNS8_CUDA_LINEAR_GATED 1u
#define RNS8_CUDA_LINEAR_MAX_K 131071
typedef struct rns8_cuda_linear_desc {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t flags; /* RNS8_CUDA_LINEAR_GATED or zero */
  int32_t device_id;
  uint32_t a_type, out_type;
  uint32_t reserved; /* must be zero */
  int64_t m, n, k, ld_a, ld_w, ld_out;
  const void* a;
  const float* a_scale; /* [m] with a_type I8, else NULL */
  const int8_t* w;
  const float* w_scale; /* [n], gated [2n] */
  const float* bias;    /* [n], gated [2n], or NULL */
  void* out;
  float* out_scale; /* [m] with out_type I8, else NULL */
  void* scratch;
  uint64_t scratch_bytes;
  uint32_t* status;
  void* stream;
} rns8_cuda_linear_desc;
/* Scratch the call needs for this descriptor (its pointers' alignments count,
 * scratch, scratch_bytes, status and stream do not); 0 for a malformed one. */
RNS8_API uint64_t rns8_cuda_linear_scratch_bytes(const rns8_cuda_linear_desc* desc);
RNS8_API rns8_status rns8_cuda_linear_device(const rns8_cuda_linear_desc* desc);
/* The kernel that a call of this descriptor runs on a GPU of sm_count
 * multiprocessors: tile = 0 with tokens on the tensor cores' lanes, else channels
 * on lanes with `tile` tokens to a tile and `splits` blocks that share k. For
 * profiles and for tests that are to cover every form. */
RNS8_API rns8_status rns8_cuda_linear_form(const rns8_cuda_linear_desc* desc, int32_t sm_count, uint32_t* tile,
                                           uint32_t* splits);

/* The step between two blocks. With N(v) = v / sqrt(mean(v^2) + eps), all in
 * 32-bit floats and rounded once on output:
 *   p     = N(y) * (weight_offset + post_weight)     (p = y without post_weight)
 *   x_out = x + scale * gate * p                     (gate = 1 without gate)
 *   h     = N(x_out) * (weight_offset + pre_weight)
 * h is written in `type` (h), as int8 rows with scales (q, q_scale; quantised
 * as above from the unrounded h), as both, or not at all (pre_weight NULL).
 * gate has `groups` rows; groups divides tokens and token t uses row
 * t / (tokens / groups). x_out may be x and h may be y. dim <= 32768. */
typedef struct rns8_cuda_residual_norm_desc {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t flags; /* must be zero */
  int32_t device_id;
  uint32_t type;        /* x, y, x_out, h: BF16, F16 or F32 */
  uint32_t weight_type; /* post_weight, pre_weight, gate: `type` or F32 */
  float scale, eps, weight_offset;
  int64_t tokens, dim, groups;
  int64_t ld_x, ld_y, ld_gate, ld_x_out, ld_h, ld_q;
  const void* x;
  const void* y;
  const void* post_weight; /* [dim] or NULL */
  const void* pre_weight;  /* [dim] or NULL */
  const void* gate;        /* [groups][dim] or NULL */
  void* x_out;
  void* h;        /* or NULL */
  int8_t* q;      /* or NULL */
  float* q_scale; /* [tokens], with q */
  void* stream;
} rns8_cuda_residual_norm_desc;
RNS8_API rns8_status rns8_cuda_residual_norm_device(const rns8_cuda_residual_norm_desc* desc);

/* Gradients of the step above from d_x_out and d_h (either may be NULL: zero),
 * the step's x_out and its input y (the row statistics are computed again):
 *   n = N(x_out), t = d_h * (weight_offset + pre_weight)
 *   d_x    = d_x_out + (t - n * mean(t * n)) / sqrt(mean(x_out^2) + eps)
 *   u = N(y), d_p = scale * gate * d_x, v = d_p * (weight_offset + post_weight)
 *   d_y    = (v - u * mean(v * u)) / sqrt(mean(y^2) + eps)
 *   d_post = sum over tokens of d_p * u, d_pre = sum over tokens of d_h * n
 *   d_gate[g] = sum over the group's tokens of scale * p * d_x
 * d_x and d_y have `type`; d_post, d_pre and d_gate are 32-bit, except that a
 * gate of one row per token (groups == tokens) has d_gate in `type`, unless
 * RNS8_CUDA_NORM_D_GATE_F32 asks for 32 bits there too (a 32-bit gate's gradient
 * then keeps its precision; weight_type F32 only). Any of the last three may be NULL. Sums over tokens run in a fixed order: equal
 * calls give equal bits. d_x may be d_x_out and d_y may be d_h. */
#define RNS8_CUDA_NORM_D_GATE_F32 2u
typedef struct rns8_cuda_residual_norm_backward_desc {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t flags; /* RNS8_CUDA_NORM_D_GATE_F32 or zero */
  int32_t device_id;
  uint32_t type;
  uint32_t weight_type;
  float scale, eps, weight_offset;
  int64_t tokens, dim, groups;
  int64_t ld_d_x_out, ld_d_h, ld_x_out, ld_y, ld_gate, ld_d_x, ld_d_y, ld_d_gate;
  const void* d_x_out;
  const void* d_h;
  const void* x_out;
  const void* y;
  const void* post_weight;
  const void* pre_weight;
  const void* gate;
  void* d_x;
  void* d_y;
  float* d_post;
  float* d_pre;
  void* d_gate;
  void* scratch;
  uint64_t scratch_bytes;
  void* stream;
} rns8_cuda_residual_norm_backward_desc;
RNS8_API uint64_t
rns8_cuda_residual_norm_backward_scratch_bytes(const rns8_cuda_residual_norm_backward_desc* desc);
RNS8_API rns8_status rns8_cuda_residual_norm_backward_device(const rns8_cuda_residual_norm_backward_desc* desc);

/* The limit of these operators' bounded device waits in SM cycles, for every
 * later call of the process: 1 to 4000000000, 0 for the usual one (the largest,
 * about two seconds). A short one shows what a wait that runs out does: a product
 * sets its status word where data was late, a norm reads the row from global
 * memory instead (at 1, every row). */
RNS8_API rns8_status rns8_cuda_quant_wait_limit(uint64_t cycles);

#ifdef __cplusplus
}
#endif

#endif /* RNS8_RNS8_QUANT_H */
