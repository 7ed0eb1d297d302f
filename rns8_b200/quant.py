"""8-bit operators of large language models on torch CUDA tensors.

    quantize_rows            rows of activations or weights -> int8 rows + scales
    gemm_scaled              int8 rows x int8 weights, a scale per row and per output channel -> float, or
                             int8 rows again for the next product
    linear                   the same from float activations, quantised per row in the call
    residual_norm            x' = x + scale * gate * N(y) and h = N(x'), differentiable
    residual_norm_quantized  the same with h as int8 rows + scales, ready for gemm_scaled
    residual_norm_backward   the gradients of residual_norm

The formulas and the treatment of zero, infinite and NaN rows are those of
include/rns8/rns8_quant.h, whose entry points these functions call. Work is
enqueued on the current stream of the tensors' device; nothing synchronises.
Inputs made on another stream are the caller's to order and to keep alive
(Tensor.record_stream), as for any torch operator. Leading dimensions of an
activation are its tokens. Bad arguments raise ValueError or TypeError before
anything is enqueued; a refusal by the library raises api.Error.
"""

from __future__ import annotations

import functools
import struct
from typing import NamedTuple

import torch

from .abi import lib
from .api import check

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_I8 = 3
_GATED = 1
MAX_K = 131071
MAX_DIM = 32768

# The descriptors of include/rns8/rns8_quant.h, packed field by field (a test
# compares them with the C compiler's layout).
QUANTIZE_DESC = struct.Struct("=QIIiI4q4Q")
LINEAR_DESC = struct.Struct("=QIIiIII6q11Q")
NORM_DESC = struct.Struct("=QIIiIIfff9q10Q")
NORM_BACKWARD_DESC = struct.Struct("=QIIiIIfff11q15Q")

_stream = torch._C._cuda_getCurrentRawStream
_status: dict[int, torch.Tensor] = {}


class QuantizedRows(NamedTuple):
    """Activations as int8 rows with a 32-bit scale each, and the type that the
    next product answers in."""

    q: torch.Tensor
    scale: torch.Tensor
    dtype: torch.dtype

    def dequantize(self) -> torch.Tensor:
        return (self.q.float() * self.scale[..., None]).to(self.dtype)


def device_status(device: int = 0) -> torch.Tensor:
    """The status word of `device`, a one-element int32 tensor that the products
    OR 0x100 into when a bounded device wait ran out."""
    word = _status.get(device)
    if word is None:
        word = _status[device] = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", device))
    return word


def check_status(device: int = 0) -> None:
    """Synchronise `device` and raise if any product on it reported a failure
    since the last check."""
    torch.cuda.synchronize(device)
    word = device_status(device)
    bits = int(word.item())
    word.zero_()
    if bits:
        raise RuntimeError(f"a bounded device wait ran out (status 0x{bits:x})")


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """t as a 2-D tensor (a view where one exists)."""
    if t.dim() == 2:
        return t
    if t.dim() == 0:
        raise ValueError(f"{name}: expected at least one dimension")
    return t.reshape(-1, t.shape[-1])


def _ld(t: torch.Tensor, name: str) -> int:
    """Leading dimension of a 2-D tensor whose rows are contiguous."""
    (rows, cols), (ld, step) = t.shape, t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{name}: elements of a row must be contiguous")
    return ld if rows > 1 else max(cols, 1)


def _float_type(t: torch.Tensor, name: str) -> int:
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: expected bfloat16, float16 or float32, got {t.dtype}")
    return code


def _cuda_device(t: torch.Tensor, name: str) -> int:
    device = t.get_device()
    if device < 0:
        raise ValueError(f"{name}: expected a CUDA tensor")
    return device


def _vector(t: torch.Tensor, size: int, device: int, name: str) -> int:
    """Address of a 32-bit vector."""
    if t.dtype != torch.float32 or t.shape != (size,) or not t.is_contiguous():
        raise TypeError(f"{name}: expected a contiguous float32 vector of {size}")
    if t.get_device() != device:
        raise ValueError(f"{name}: expected a tensor on cuda:{device}")
    return t.data_ptr()


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) with x ~ q * scale[..., None]: int8 rows and one 32-bit scale
    per row. Rows of q start on 16-byte boundaries (its leading dimension is
    padded where the row length is not a multiple of 16)."""
    code = _float_type(x, "x")
    device = _cuda_device(x, "x")
    shape = x.shape
    x = _rows(x, "x")
    rows, cols = x.shape
    if cols == 0:
        raise ValueError("x: rows are empty")
    ld = (cols + 15) // 16 * 16
    q = x.new_empty((rows, ld), dtype=torch.int8)
    scale = x.new_empty(rows, dtype=torch.float32)
    desc = QUANTIZE_DESC.pack(QUANTIZE_DESC.size, 1, 0, device, code, rows, cols, _ld(x, "x"), ld, x.data_ptr(),
                              q.data_ptr(), scale.data_ptr(), _stream(device))
    status = lib().rns8_cuda_quantize_rows_device(desc)
    if status:
        check(status, "rns8_cuda_quantize_rows_device")
    if ld != cols:
        q = q[:, :cols]
    if len(shape) == 2:
        return q, scale
    if len(shape) == 1:
        return q[0], scale[0]
    return q.unflatten(0, shape[:-1]), scale.view(shape[:-1])


@functools.lru_cache(maxsize=4096)
def _linear_scratch(device, flags, a_type, out_type, m, n, k, ld_a, ld_w, align_a, align_w):
    # Pointers stand for their alignments only: the query reads no memory.
    desc = LINEAR_DESC.pack(LINEAR_DESC.size, 1, flags, device, a_type, out_type, 0, m, n, k, ld_a, ld_w, n,
                            4096 + align_a, 4096 if a_type == _I8 else 0, 4096 + align_w, 4096, 0, 4096,
                            4096 if out_type == _I8 else 0, 0, 0, 0, 0)
    return lib().rns8_cuda_linear_scratch_bytes(desc)


def _linear(a, a_type, a_scale, device, w, w_scale, bias, gated, out_dtype, quantize):
    lead = a.shape[:-1]
    if len(lead) != 1:
        a = _rows(a, "activations")
    if w.dtype != torch.int8 or w.dim() != 2:
        raise TypeError("w: expected a 2-D int8 tensor (output channels x inputs)")
    m, k = a.shape
    rows, wk = w.shape
    if wk != k:
        raise ValueError(f"w: expected rows of {k}, got {wk}")
    if gated and rows % 2:
        raise ValueError("w: a gated product needs an even number of rows (gate rows, then up rows)")
    n = rows // 2 if gated else rows
    if n == 0 or k == 0:
        raise ValueError("w: empty")
    if w.get_device() != device:
        raise ValueError(f"w: expected a tensor on cuda:{device}")
    p_scale = _vector(w_scale, rows, device, "w_scale")
    p_bias = _vector(bias, rows, device, "bias") if bias is not None else 0
    out_type = _TYPES.get(out_dtype)
    if out_type is None:
        raise TypeError(f"out_dtype: expected bfloat16, float16 or float32, got {out_dtype}")
    out_scale, ld_out, p_out_scale = None, n, 0
    if quantize:
        out_type, ld_out = _I8, (n + 15) // 16 * 16
        out = a.new_empty((m, ld_out), dtype=torch.int8)
        out_scale = a.new_empty(m, dtype=torch.float32)
        p_out_scale = out_scale.data_ptr()
    else:
        out = a.new_empty((m, n), dtype=out_dtype)
    if m:
        flags = _GATED if gated else 0
        ld_a, ld_w, pa, pw = _ld(a, "activations"), _ld(w, "w"), a.data_ptr(), w.data_ptr()
        need = _linear_scratch(device, flags, a_type, out_type, m, n, k, ld_a, ld_w, pa & 15, pw & 15)
        scratch = a.new_empty(need, dtype=torch.uint8) if need else None
        desc = LINEAR_DESC.pack(LINEAR_DESC.size, 1, flags, device, a_type, out_type, 0, m, n, k, ld_a, ld_w, ld_out, pa,
                                a_scale, pw, p_scale, p_bias, out.data_ptr(), p_out_scale,
                                scratch.data_ptr() if need else 0, need, device_status(device).data_ptr(),
                                _stream(device))
        status = lib().rns8_cuda_linear_device(desc)
        if status:
            check(status, "rns8_cuda_linear_device")
    if quantize:
        if ld_out != n:
            out = out[:, :n]
        if len(lead) != 1:
            out, out_scale = (out.unflatten(0, lead), out_scale.view(lead)) if lead else (out[0], out_scale[0])
        return QuantizedRows(out, out_scale, out_dtype)
    return out if len(lead) == 1 else out.view(*lead, n)


def gemm_scaled(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, gated: bool = False, out_dtype: torch.dtype = torch.bfloat16,
                quantize: bool | None = None):
    """(a @ w.T) * a_scale[..., None] * w_scale + bias from int8 a (tokens x k)
    and int8 w (output channels x k), summed exactly in 32-bit integers. With
    gated, w's first half are the gate's channels: silu(first) * second.

    The result is a tensor of out_dtype, or, with quantize, QuantizedRows made
    from the 32-bit values: int8 in, int8 out, for a chain of products. A gated
    product's result is the next product's tokens, so there quantize is the
    default; pass quantize=False for a tensor."""
    if a.dtype != torch.int8:
        raise TypeError(f"a: expected int8, got {a.dtype}")
    if a_scale.dtype != torch.float32 or a_scale.shape != a.shape[:-1] or not a_scale.is_contiguous():
        raise TypeError("a_scale: expected a contiguous float32 tensor with one value per row of a")
    device = _cuda_device(a, "a")
    if a_scale.get_device() != device:
        raise ValueError("a_scale: expected a tensor on a's device")
    return _linear(a, _I8, a_scale.data_ptr(), device, w, w_scale, bias, gated, out_dtype,
                   gated if quantize is None else quantize)


def linear(x: torch.Tensor | QuantizedRows, w: torch.Tensor, w_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
           gated: bool = False, out_dtype: torch.dtype | None = None, quantize: bool = False):
    """gemm_scaled(*quantize_rows(x), w, w_scale) in one call; the result has
    x's type unless out_dtype is given. QuantizedRows go in as they are."""
    if isinstance(x, QuantizedRows):
        return gemm_scaled(x.q, x.scale, w, w_scale, bias=bias, gated=gated, out_dtype=out_dtype or x.dtype,
                           quantize=quantize)
    code = _float_type(x, "x")
    return _linear(x, code, 0, _cuda_device(x, "x"), w, w_scale, bias, gated, out_dtype or x.dtype, quantize)


def _norm_weights(x, device, tokens, dim, post_weight, pre_weight, gate):
    """(weight type, groups, gate's leading dimension, post, pre, gate addresses)
    of a norm's checked parameters."""
    dtype, post, pre, p_gate, groups, ld_gate = None, 0, 0, 0, 1, dim
    if post_weight is not None:
        dtype, post = post_weight.dtype, post_weight.data_ptr()
        if post_weight.shape != (dim,) or not post_weight.is_contiguous() or post_weight.get_device() != device:
            raise ValueError(f"post_weight: expected a contiguous vector of {dim} on cuda:{device}")
    if pre_weight is not None:
        pre = pre_weight.data_ptr()
        if pre_weight.shape != (dim,) or not pre_weight.is_contiguous() or pre_weight.get_device() != device:
            raise ValueError(f"pre_weight: expected a contiguous vector of {dim} on cuda:{device}")
        if dtype is not None and pre_weight.dtype != dtype:
            raise TypeError("pre_weight: the weights and the gate share one type")
        dtype = pre_weight.dtype
    if gate is not None:
        groups, gate_dim = gate.shape
        if gate_dim != dim or gate.get_device() != device:
            raise ValueError(f"gate: expected rows of {dim} on cuda:{device}")
        if dtype is not None and gate.dtype != dtype:
            raise TypeError("gate: the weights and the gate share one type")
        if tokens and (groups == 0 or tokens % groups):
            raise ValueError(f"gate: {groups} rows do not divide {tokens} tokens")
        dtype, ld_gate, p_gate = gate.dtype, _ld(gate, "gate"), gate.data_ptr()
    if dtype is None:
        dtype = x.dtype
    elif dtype != x.dtype and dtype != torch.float32:
        raise TypeError(f"weights: expected {x.dtype} or float32, got {dtype}")
    return _TYPES[dtype], groups, ld_gate, post, pre, p_gate


def _norm_rows(x, y, name):
    """Type, device, sizes and 2-D forms of a norm's two activations."""
    code = _float_type(x, name)
    device = _cuda_device(x, name)
    if y.shape != x.shape or y.dtype != x.dtype:
        raise ValueError(f"y: expected {name}'s type and shape")
    if y.get_device() != device:
        raise ValueError(f"y: expected a tensor on cuda:{device}")
    x, y = _rows(x, name), _rows(y, "y")
    tokens, dim = x.shape
    if not 0 < dim <= MAX_DIM:
        raise ValueError(f"{name}: rows must have 1 to {MAX_DIM} elements")
    return code, device, tokens, dim, x, y


def _norm_forward(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset, want_h, want_q):
    shape = x.shape
    code, device, tokens, dim, x, y = _norm_rows(x, y, "x")
    if gate is not None:
        gate = _rows(gate, "gate")
    wcode, groups, ld_gate, post, pre, p_gate = _norm_weights(x, device, tokens, dim, post_weight, pre_weight, gate)
    x_out = x.new_empty((tokens, dim))
    h = x.new_empty((tokens, dim)) if want_h else None
    ld_q, q, s = (dim + 15) // 16 * 16, None, None
    if want_q:
        q = x.new_empty((tokens, ld_q), dtype=torch.int8)
        s = x.new_empty(tokens, dtype=torch.float32)
    if tokens:
        desc = NORM_DESC.pack(NORM_DESC.size, 1, 0, device, code, wcode, scale, eps, weight_offset, tokens, dim, groups,
                              _ld(x, "x"), _ld(y, "y"), ld_gate, dim, dim, ld_q, x.data_ptr(), y.data_ptr(), post, pre,
                              p_gate, x_out.data_ptr(), h.data_ptr() if want_h else 0, q.data_ptr() if want_q else 0,
                              s.data_ptr() if want_q else 0, _stream(device))
        status = lib().rns8_cuda_residual_norm_device(desc)
        if status:
            check(status, "rns8_cuda_residual_norm_device")
    if want_q and ld_q != dim:
        q = q[:, :dim]
    if len(shape) == 2:
        return x_out, h, q, s
    lead = shape[:-1]
    if want_q:
        q = q.unflatten(0, lead) if lead else q[0]
        s = s.view(lead)
    return x_out.view(shape), h.view(shape) if want_h else None, q, s


@functools.lru_cache(maxsize=4096)
def _backward_scratch(device, code, wcode, tokens, dim, groups, post, pre, gate):
    # Sizes and which gradients are wanted decide: the query reads no memory.
    desc = NORM_BACKWARD_DESC.pack(NORM_BACKWARD_DESC.size, 1, 0, device, code, wcode, 1.0, 1.0, 0.0, tokens, dim, groups,
                                   *(dim,) * 8, 4096, 4096, 4096, 4096, 4096 * post, 4096 * pre, 4096 * gate, 4096, 4096,
                                   4096 * post, 4096 * pre, 4096 * gate, 0, 0, 0)
    return lib().rns8_cuda_residual_norm_backward_scratch_bytes(desc)


def residual_norm_backward(d_x_out: torch.Tensor | None, d_h: torch.Tensor | None, x_out: torch.Tensor, y: torch.Tensor, *,
                           post_weight: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None,
                           gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-6,
                           weight_offset: float = 0.0):
    """(d_x, d_y, d_post_weight, d_pre_weight, d_gate) of residual_norm from the
    gradients of its two results, its first result x_out and its input y. The
    sums over tokens are 32-bit; d_gate is x's type where the gate has one row
    per token. Entries without their input are None."""
    shape = x_out.shape
    gate_shape = gate.shape if gate is not None else None
    code, device, tokens, dim, x_out, y = _norm_rows(x_out, y, "x_out")
    if gate is not None:
        gate = _rows(gate, "gate")
    wcode, groups, ld_gate, post, pre, p_gate = _norm_weights(x_out, device, tokens, dim, post_weight, pre_weight, gate)
    p_dxo = p_dh = 0
    ld_dxo = ld_dh = dim
    if d_x_out is not None:
        if d_x_out.shape != shape or d_x_out.dtype != x_out.dtype or d_x_out.get_device() != device:
            raise ValueError("d_x_out: expected x_out's type, shape and device")
        d_x_out = _rows(d_x_out, "d_x_out")
        p_dxo, ld_dxo = d_x_out.data_ptr(), _ld(d_x_out, "d_x_out")
    if d_h is not None:
        if d_h.shape != shape or d_h.dtype != x_out.dtype or d_h.get_device() != device:
            raise ValueError("d_h: expected x_out's type, shape and device")
        d_h = _rows(d_h, "d_h")
        p_dh, ld_dh = d_h.data_ptr(), _ld(d_h, "d_h")
    d_x = x_out.new_empty((tokens, dim))
    d_y = x_out.new_empty((tokens, dim))
    d_post = d_pre = d_gate = None
    if post and pre:
        d_post, d_pre = x_out.new_empty((2, dim), dtype=torch.float32).unbind(0)
    elif post:
        d_post = x_out.new_empty(dim, dtype=torch.float32)
    elif pre:
        d_pre = x_out.new_empty(dim, dtype=torch.float32)
    if gate is not None:
        d_gate = x_out.new_empty((groups, dim), dtype=x_out.dtype if groups == tokens else torch.float32)
    need = _backward_scratch(device, code, wcode, tokens, dim, groups, post != 0, pre != 0, gate is not None)
    scratch = x_out.new_empty(need, dtype=torch.uint8) if need else None
    desc = NORM_BACKWARD_DESC.pack(
        NORM_BACKWARD_DESC.size, 1, 0, device, code, wcode, scale, eps, weight_offset, tokens, dim, groups, ld_dxo, ld_dh,
        _ld(x_out, "x_out"), _ld(y, "y"), ld_gate, dim, dim, dim, p_dxo, p_dh, x_out.data_ptr(), y.data_ptr(), post, pre,
        p_gate, d_x.data_ptr(), d_y.data_ptr(), d_post.data_ptr() if post else 0, d_pre.data_ptr() if pre else 0,
        d_gate.data_ptr() if gate is not None else 0, scratch.data_ptr() if need else 0, need, _stream(device))
    status = lib().rns8_cuda_residual_norm_backward_device(desc)
    if status:
        check(status, "rns8_cuda_residual_norm_backward_device")
    if len(shape) != 2:
        d_x, d_y = d_x.view(shape), d_y.view(shape)
    if gate is not None and len(gate_shape) != 2:
        d_gate = d_gate.view(gate_shape)
    return d_x, d_y, d_post, d_pre, d_gate


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_weight, pre_weight, gate, scale, eps, weight_offset):
        x_out, h, _, _ = _norm_forward(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset,
                                       pre_weight is not None, False)
        ctx.save_for_backward(x_out, y, post_weight, pre_weight, gate)
        ctx.params = (scale, eps, weight_offset)
        ctx.set_materialize_grads(False)
        return x_out, h

    @staticmethod
    def backward(ctx, d_x_out, d_h):
        x_out, y, post_weight, pre_weight, gate = ctx.saved_tensors
        scale, eps, weight_offset = ctx.params
        if d_x_out is None and d_h is None:
            return (None,) * 8
        d_x, d_y, d_post, d_pre, d_gate = residual_norm_backward(
            d_x_out.contiguous() if d_x_out is not None else None, d_h.contiguous() if d_h is not None else None, x_out, y,
            post_weight=post_weight, pre_weight=pre_weight, gate=gate, scale=scale, eps=eps, weight_offset=weight_offset)

        def cast(g, like):
            return None if g is None else g.to(like.dtype)

        return d_x, d_y, cast(d_post, post_weight), cast(d_pre, pre_weight), cast(d_gate, gate), None, None, None


def residual_norm(x: torch.Tensor, y: torch.Tensor, *, post_weight: torch.Tensor | None = None,
                  pre_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
                  eps: float = 1e-6, weight_offset: float = 0.0):
    """(x_out, h): x_out = x + scale * gate * N(y), h = N(x_out), where N divides
    by the row's root mean square and multiplies by weight_offset + weight
    (post_weight for y, pre_weight for h). Without post_weight y enters as it
    is; without pre_weight h is None. gate is one row of channels or rows that
    each serve an equal run of tokens. Gradients flow to every tensor."""
    if torch.is_grad_enabled():
        tensors = (x, y, post_weight, pre_weight, gate)
        if any([t is not None and t.requires_grad for t in tensors]):
            return _ResidualNorm.apply(*tensors, scale, eps, weight_offset)
    return _norm_forward(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset, pre_weight is not None, False)[:2]


def residual_norm_quantized(x: torch.Tensor, y: torch.Tensor, *, pre_weight: torch.Tensor,
                            post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                            scale: float = 1.0, eps: float = 1e-6, weight_offset: float = 0.0):
    """(x_out, q, q_scale): residual_norm with h quantised per row as
    quantize_rows does, from its unrounded values. For inference: no gradient."""
    x_out, _, q, s = _norm_forward(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset, False, True)
    return x_out, q, s
