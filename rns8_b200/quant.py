"""8-bit operators of large language models on torch CUDA tensors.

    quantize_rows            rows of activations or weights -> int8 rows + scales
    gemm_scaled              int8 rows x int8 weights -> float, a scale per row and per output channel
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
LINEAR_DESC = struct.Struct("=QIIiIII6q10Q")
NORM_DESC = struct.Struct("=QIIiIIfff9q10Q")
NORM_BACKWARD_DESC = struct.Struct("=QIIiIIfff11q15Q")

_stream = torch._C._cuda_getCurrentRawStream
_status: dict[int, torch.Tensor] = {}


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
    """t as a 2-D tensor with contiguous rows."""
    if t.dim() != 2:
        if t.dim() == 0:
            raise ValueError(f"{name}: expected at least one dimension")
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name}: elements of a row must be contiguous")
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _same_device(device: int, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.get_device() != device:
            raise ValueError(f"{name}: expected a tensor on cuda:{device}")


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
    q = torch.empty((rows, ld), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    desc = QUANTIZE_DESC.pack(QUANTIZE_DESC.size, 1, 0, device, code, rows, cols, _ld(x), ld, x.data_ptr(), q.data_ptr(),
                              scale.data_ptr(), _stream(device))
    check(lib().rns8_cuda_quantize_rows_device(desc), "rns8_cuda_quantize_rows_device")
    if len(shape) == 1:
        return q[0, :cols], scale[0]
    return q[:, :cols].unflatten(0, shape[:-1]) if len(shape) > 2 else q[:, :cols], scale.view(shape[:-1])


@functools.lru_cache(maxsize=1024)
def _linear_scratch(device, flags, a_type, out_type, m, n, k, ld_a, ld_w, ld_out, align_a, align_w, has_bias):
    # Pointers stand for their alignments only: the query reads no memory.
    desc = LINEAR_DESC.pack(LINEAR_DESC.size, 1, flags, device, a_type, out_type, 0, m, n, k, ld_a, ld_w, ld_out,
                            4096 + align_a, 4096 if a_type == _I8 else 0, 4096 + align_w, 4096, 4096 * has_bias, 4096, 0,
                            0, 0, 0)
    return lib().rns8_cuda_linear_scratch_bytes(desc)


def _linear(a, a_type, a_scale, w, w_scale, bias, gated, out_dtype):
    device = _cuda_device(a, "activations")
    lead = a.shape[:-1]
    a = _rows(a, "activations")
    if w.dtype != torch.int8 or w.dim() != 2:
        raise TypeError("w: expected a 2-D int8 tensor (output channels x inputs)")
    w = _rows(w, "w")
    m, k = a.shape
    rows, wk = w.shape
    if wk != k:
        raise ValueError(f"w: expected rows of {k}, got {wk}")
    if gated and rows % 2:
        raise ValueError("w: a gated product needs an even number of rows (gate rows, then up rows)")
    n = rows // 2 if gated else rows
    if n == 0 or k == 0:
        raise ValueError("w: empty")
    if w_scale.dtype != torch.float32 or w_scale.shape != (rows,) or not w_scale.is_contiguous():
        raise TypeError(f"w_scale: expected a contiguous float32 vector of {rows}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (rows,) or not bias.is_contiguous()):
        raise TypeError(f"bias: expected a contiguous float32 vector of {rows}")
    _same_device(device, w=w, w_scale=w_scale, bias=bias)
    out_type = _TYPES.get(out_dtype)
    if out_type is None:
        raise TypeError(f"out_dtype: expected bfloat16, float16 or float32, got {out_dtype}")
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if m:
        flags = _GATED if gated else 0
        ld_a, ld_w, pa, pw = _ld(a), _ld(w), a.data_ptr(), w.data_ptr()
        need = _linear_scratch(device, flags, a_type, out_type, m, n, k, ld_a, ld_w, n, pa & 15, pw & 15,
                               bias is not None)
        scratch = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None
        desc = LINEAR_DESC.pack(LINEAR_DESC.size, 1, flags, device, a_type, out_type, 0, m, n, k, ld_a, ld_w, n, pa,
                                a_scale.data_ptr() if a_scale is not None else 0, pw, w_scale.data_ptr(),
                                bias.data_ptr() if bias is not None else 0, out.data_ptr(),
                                scratch.data_ptr() if need else 0, need, device_status(device).data_ptr(),
                                _stream(device))
        check(lib().rns8_cuda_linear_device(desc), "rns8_cuda_linear_device")
    return out if len(lead) == 1 else out.view(*lead, n)


def gemm_scaled(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, gated: bool = False,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(a @ w.T) * a_scale[..., None] * w_scale + bias from int8 a (tokens x k)
    and int8 w (output channels x k), summed exactly in 32-bit integers. With
    gated, w's first half are the gate's channels: silu(first) * second."""
    if a.dtype != torch.int8:
        raise TypeError(f"a: expected int8, got {a.dtype}")
    if a_scale.dtype != torch.float32 or a_scale.shape != a.shape[:-1] or not a_scale.is_contiguous():
        raise TypeError("a_scale: expected a contiguous float32 tensor with one value per row of a")
    if a_scale.get_device() != a.get_device():
        raise ValueError("a_scale: expected a tensor on a's device")
    return _linear(a, _I8, a_scale, w, w_scale, bias, gated, out_dtype)


def linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
           gated: bool = False, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """gemm_scaled(*quantize_rows(x), w, w_scale) in one call; the result has
    x's type unless out_dtype is given."""
    return _linear(x, _float_type(x, "x"), None, w, w_scale, bias, gated, out_dtype or x.dtype)


class _NormArgs:
    """Checked arguments shared by the forward and backward calls."""

    __slots__ = ("device", "code", "wcode", "tokens", "dim", "groups", "ld_gate", "post", "pre", "gate")

    def __init__(self, x, y, post_weight, pre_weight, gate):
        self.code = _float_type(x, "x")
        self.device = device = _cuda_device(x, "x")
        if y.dtype != x.dtype or y.shape != x.shape:
            raise ValueError("y: expected x's type and shape")
        self.tokens, self.dim = x.shape
        if not 0 < self.dim <= MAX_DIM:
            raise ValueError(f"x: rows must have 1 to {MAX_DIM} elements")
        wdtype = None
        for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
            if w is None:
                continue
            if w.shape != (self.dim,) or not w.is_contiguous():
                raise ValueError(f"{name}: expected a contiguous vector of {self.dim}")
            if wdtype is not None and w.dtype != wdtype:
                raise TypeError(f"{name}: the weights and the gate share one type")
            wdtype = w.dtype
        self.groups, self.ld_gate, self.gate = 1, self.dim, 0
        if gate is not None:
            if gate.shape[1] != self.dim:
                raise ValueError(f"gate: expected rows of {self.dim}")
            if wdtype is not None and gate.dtype != wdtype:
                raise TypeError("gate: the weights and the gate share one type")
            wdtype = gate.dtype
            self.groups = gate.shape[0]
            if self.tokens and (self.groups == 0 or self.tokens % self.groups):
                raise ValueError(f"gate: {self.groups} rows do not divide {self.tokens} tokens")
            self.ld_gate, self.gate = _ld(gate), gate.data_ptr()
        if wdtype is not None and wdtype not in (x.dtype, torch.float32):
            raise TypeError(f"weights: expected {x.dtype} or float32, got {wdtype}")
        self.wcode = self.code if wdtype is None else _TYPES[wdtype]
        _same_device(device, y=y, post_weight=post_weight, pre_weight=pre_weight, gate=gate)
        self.post = post_weight.data_ptr() if post_weight is not None else 0
        self.pre = pre_weight.data_ptr() if pre_weight is not None else 0


def _norm_forward(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset, want_h, want_q):
    shape = x.shape
    if y.shape != shape:
        raise ValueError("y: expected x's shape")
    x, y = _rows(x, "x"), _rows(y, "y")
    gate = _rows(gate, "gate") if gate is not None else None
    a = _NormArgs(x, y, post_weight, pre_weight, gate)
    x_out = torch.empty((a.tokens, a.dim), dtype=x.dtype, device=x.device)
    h = torch.empty((a.tokens, a.dim), dtype=x.dtype, device=x.device) if want_h else None
    ld_q = (a.dim + 15) // 16 * 16
    q = torch.empty((a.tokens, ld_q), dtype=torch.int8, device=x.device) if want_q else None
    s = torch.empty(a.tokens, dtype=torch.float32, device=x.device) if want_q else None
    if a.tokens:
        desc = NORM_DESC.pack(NORM_DESC.size, 1, 0, a.device, a.code, a.wcode, scale, eps, weight_offset, a.tokens, a.dim,
                              a.groups, _ld(x), _ld(y), a.ld_gate, a.dim, a.dim, ld_q, x.data_ptr(), y.data_ptr(),
                              a.post, a.pre, a.gate, x_out.data_ptr(), h.data_ptr() if want_h else 0,
                              q.data_ptr() if want_q else 0, s.data_ptr() if want_q else 0, _stream(a.device))
        check(lib().rns8_cuda_residual_norm_device(desc), "rns8_cuda_residual_norm_device")
    if len(shape) == 2:
        return x_out, h, q[:, :a.dim] if want_q else None, s
    lead = shape[:-1]
    return (x_out.view(shape), h.view(shape) if want_h else None,
            (q[0, :a.dim] if len(lead) == 0 else q[:, :a.dim].unflatten(0, lead)) if want_q else None,
            s.view(lead) if want_q else None)


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
    x_out, y = _rows(x_out, "x_out"), _rows(y, "y")
    gate = _rows(gate, "gate") if gate is not None else None
    a = _NormArgs(x_out, y, post_weight, pre_weight, gate)
    grads = []
    for name, g in (("d_x_out", d_x_out), ("d_h", d_h)):
        if g is not None:
            if g.shape != shape or g.dtype != x_out.dtype:
                raise ValueError(f"{name}: expected x_out's type and shape")
            _same_device(a.device, **{name: g})
            g = _rows(g, name)
        grads.append(g)
    dxo, dh = grads
    dev, t, dim = x_out.device, a.tokens, a.dim
    d_x = torch.empty((t, dim), dtype=x_out.dtype, device=dev)
    d_y = torch.empty((t, dim), dtype=x_out.dtype, device=dev)
    d_post = torch.empty(dim, dtype=torch.float32, device=dev) if post_weight is not None else None
    d_pre = torch.empty(dim, dtype=torch.float32, device=dev) if pre_weight is not None else None
    d_gate = None
    if gate is not None:
        d_gate = torch.empty((a.groups, dim), dtype=x_out.dtype if a.groups == t else torch.float32, device=dev)

    def pack(scratch, size):
        return NORM_BACKWARD_DESC.pack(
            NORM_BACKWARD_DESC.size, 1, 0, a.device, a.code, a.wcode, scale, eps, weight_offset, t, dim, a.groups,
            _ld(dxo) if dxo is not None else dim, _ld(dh) if dh is not None else dim, _ld(x_out), _ld(y), a.ld_gate, dim,
            dim, dim, dxo.data_ptr() if dxo is not None else 0, dh.data_ptr() if dh is not None else 0,
            x_out.data_ptr(), y.data_ptr(), a.post, a.pre, a.gate, d_x.data_ptr(), d_y.data_ptr(),
            d_post.data_ptr() if d_post is not None else 0, d_pre.data_ptr() if d_pre is not None else 0,
            d_gate.data_ptr() if d_gate is not None else 0, scratch, size, _stream(a.device))

    handle = lib()
    need = handle.rns8_cuda_residual_norm_backward_scratch_bytes(pack(0, 0))
    scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    check(handle.rns8_cuda_residual_norm_backward_device(pack(scratch.data_ptr() if need else 0, need)),
          "rns8_cuda_residual_norm_backward_device")
    return (d_x.view(shape), d_y.view(shape), d_post, d_pre, d_gate.view(gate_shape) if gate is not None else None)


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
    tensors = (x, y, post_weight, pre_weight, gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _ResidualNorm.apply(*tensors, scale, eps, weight_offset)
    return _norm_forward(*tensors, scale, eps, weight_offset, pre_weight is not None, False)[:2]


def residual_norm_quantized(x: torch.Tensor, y: torch.Tensor, *, pre_weight: torch.Tensor,
                            post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                            scale: float = 1.0, eps: float = 1e-6, weight_offset: float = 0.0):
    """(x_out, q, q_scale): residual_norm with h quantised per row as
    quantize_rows does, from its unrounded values. For inference: no gradient."""
    x_out, _, q, s = _norm_forward(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset, False, True)
    return x_out, q, s
