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
activation are its tokens; rows that share memory (expand) are copied first.

residual_norm alone has a derivative. The others are for inference: asking for a
gradient through their results raises RuntimeError, a forward-mode tangent among
their inputs NotImplementedError. Bad arguments raise ValueError or TypeError
before anything is enqueued; a refusal by the library raises api.Error.
"""

from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import threading
from typing import NamedTuple

import torch

from . import abi
from .api import check

MAX_K = 131071
MAX_DIM = 32768


class QuantizedRows(NamedTuple):
    """Activations as int8 rows with a 32-bit scale each, and the type that the
    next product answers in."""

    q: torch.Tensor
    scale: torch.Tensor
    dtype: torch.dtype

    def dequantize(self) -> torch.Tensor:
        return (self.q.float() * self.scale[..., None]).to(self.dtype)


_status: dict[int, torch.Tensor] = {}
_status_lock = threading.RLock()


def device_status(device: int = 0) -> torch.Tensor:
    """The status word of `device`, a one-element int32 tensor that the products
    OR 0x100 into when a bounded device wait ran out. The first call on a device
    allocates it, so that call cannot be part of a stream capture."""
    word = _status.get(device)
    if word is not None:
        return word
    # One word for the process's life: the binding keeps its address, and an
    # allocation lets other threads run.
    with _status_lock:
        if device not in _status:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first product on a device cannot be captured: run one, or device_status(), before")
            word = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", device))
            torch.cuda.current_stream(device).synchronize()  # other streams may use it next
            _status.setdefault(device, word)
        return _status[device]


def check_status(device: int = 0) -> None:
    """Synchronise `device` and raise if any product on it reported a failure
    since the last check."""
    torch.cuda.synchronize(device)
    word = device_status(device)
    bits = int(word.item())
    if bits:
        word.zero_()
        torch.cuda.synchronize(device)  # a product on another stream may report from here on
        raise RuntimeError(f"a bounded device wait ran out (status 0x{bits:x})")


def _load_binding():
    """The compiled torch binding (csrc/torch/quant_torch.cpp), bound to the
    library that abi.lib() loads. Raises where it has not been built."""
    path = abi.PKG / "_build" / "_quant_torch.so"
    if not path.exists():
        raise RuntimeError(f"{path} is missing: build it with `python -m rns8_b200.build`")
    loader = importlib.machinery.ExtensionFileLoader("_quant_torch", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_quant_torch", loader))
    loader.exec_module(module)
    lib = abi.lib()
    names = ("quantize_rows_device", "linear_scratch_bytes", "linear_device", "residual_norm_device",
             "residual_norm_backward_scratch_bytes", "residual_norm_backward_device")
    module.bind(*(C.cast(getattr(lib, f"rns8_cuda_{n}"), C.c_void_p).value for n in names), check,
                lambda device: device_status(device).data_ptr(), torch.OutOfMemoryError)
    return module


_binding = _load_binding()


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) with x ~ q * scale[..., None]: int8 rows and one 32-bit scale
    per row. Rows of q start on 16-byte boundaries (its leading dimension is
    padded where the row length is not a multiple of 16)."""
    return _binding.quantize_rows(x)


def gemm_scaled(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, gated: bool = False, out_dtype: torch.dtype = torch.bfloat16,
                quantize: bool | None = None):
    """(a @ w.T) * a_scale[..., None] * w_scale + bias from int8 a (tokens x k)
    and int8 w (output channels x k), summed exactly in 32-bit integers. With
    gated, w's first half are the gate's channels: silu(first) * second.

    The result is a tensor of out_dtype, or, with quantize, QuantizedRows made
    from the 32-bit values: int8 in, int8 out, for a chain of products, whose next
    product then answers in out_dtype. quantize unset means: as the next step
    takes it, QuantizedRows from a gated product, a tensor from any other. Say
    quantize=True or False where the result's type matters to the caller."""
    if a_scale is None:
        raise TypeError("a_scale: expected a tensor")
    if quantize or (quantize is None and gated):
        return QuantizedRows(*_binding.linear(a, a_scale, w, w_scale, bias, bool(gated), out_dtype, True), out_dtype)
    return _binding.linear(a, a_scale, w, w_scale, bias, bool(gated), out_dtype, False)


def linear(x: torch.Tensor | QuantizedRows, w: torch.Tensor, w_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
           gated: bool = False, out_dtype: torch.dtype | None = None, quantize: bool = False):
    """gemm_scaled(*quantize_rows(x), w, w_scale, quantize=quantize) in one call:
    float rows in and, gated or not, a tensor out, in x's type unless out_dtype is
    given; QuantizedRows with quantize. QuantizedRows go in as they are."""
    if isinstance(x, QuantizedRows):
        return gemm_scaled(x.q, x.scale, w, w_scale, bias=bias, gated=gated, out_dtype=out_dtype or x.dtype,
                           quantize=bool(quantize))
    if quantize:
        return QuantizedRows(*_binding.linear(x, None, w, w_scale, bias, bool(gated), out_dtype, True),
                             out_dtype or x.dtype)
    return _binding.linear(x, None, w, w_scale, bias, bool(gated), out_dtype, False)


def residual_norm_backward(d_x_out: torch.Tensor | None, d_h: torch.Tensor | None, x_out: torch.Tensor,
                           y: torch.Tensor, *, post_weight: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None,
                           gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-6,
                           weight_offset: float = 0.0):
    """(d_x, d_y, d_post_weight, d_pre_weight, d_gate) of residual_norm from the
    gradients of its two results, its first result x_out and its input y. The
    sums over tokens are 32-bit; the d_gate of a gate in x's type with one row
    per token is in that type. Entries without their input are None."""
    return _binding.residual_norm_backward(d_x_out, d_h, x_out, y, post_weight, pre_weight, gate, scale, eps,
                                           weight_offset)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_weight, pre_weight, gate, scale, eps, weight_offset):
        x_out, h = _binding.residual_norm(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset, 1)
        ctx.save_for_backward(x_out, y, post_weight, pre_weight, gate)
        ctx.params = (scale, eps, weight_offset)
        ctx.set_materialize_grads(False)
        return x_out, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_x_out, d_h):
        x_out, y, post_weight, pre_weight, gate = ctx.saved_tensors
        if d_x_out is None and d_h is None:
            return (None,) * 8
        d_x, d_y, d_post, d_pre, d_gate = _binding.residual_norm_backward(
            d_x_out.contiguous() if d_x_out is not None else None, d_h.contiguous() if d_h is not None else None,
            x_out, y, post_weight, pre_weight, gate, *ctx.params)

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
    each serve an equal run of tokens. Gradients flow to every tensor;
    forward-mode tangents are refused (NotImplementedError)."""
    out = _binding.residual_norm(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset, 0)
    if out is None:  # a derivative is wanted
        return _ResidualNorm.apply(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset)
    return out


def residual_norm_quantized(x: torch.Tensor, y: torch.Tensor, *, pre_weight: torch.Tensor,
                            post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                            scale: float = 1.0, eps: float = 1e-6, weight_offset: float = 0.0):
    """(x_out, q, q_scale): residual_norm with h quantised per row as
    quantize_rows does, from its unrounded values. For inference: no derivative."""
    return _binding.residual_norm(x, y, post_weight, pre_weight, gate, scale, eps, weight_offset, 2)
