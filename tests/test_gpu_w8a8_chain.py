"""The chain norm -> int8 rows -> gated product -> int8 rows -> product against
its definition in 64 bits, each step from the rows that the step before gave.

A 32-bit value near the middle between two int8 steps may round the other way
than the 64-bit one. With E a bound on the error of the values before a
quantisation (scale s, largest magnitude top), its scale differs by the factor
r = max E / top + 4 u32, and its int8 value where the 64-bit quotient is within
E / s + 128 r of a middle. E is what test_gpu_residual_norm and
test_gpu_quant_linear allow the 32-bit operations."""

import importlib.util
from pathlib import Path

import pytest

from test_gpu_quant_linear import check_close, linear_ref, rng
from test_gpu_residual_norm import EPS32, close, forward_ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def check_rows(q, scale, v, err):
    """int8 rows are the quantisation of the 64-bit values v but for turns."""
    top = v.abs().amax(1, keepdim=True)
    quotient = v / (top / 127)
    r = err.amax(1, keepdim=True) / top + 4 * EPS32
    assert bool(((scale.double()[:, None] - top / 127).abs() <= r * top / 127).all())
    reach = err / (top / 127) + 128 * r
    assert float(reach.max()) < 0.5
    turns = (quotient - torch.floor(quotient) - 0.5).abs() <= reach
    off = (q - torch.round(quotient)).abs()
    assert bool(((off == 0) | (turns & (off == 1))).all())
    assert float(turns.double().mean()) < 0.01  # so that the comparison says something


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,dim,hidden", [(1, 256, 512), (7, 512, 328), (48, 1024, 2048), (300, 520, 1000),
                                               (1300, 1024, 2048)])
def test_chain(tokens, dim, hidden, dtype):
    from rns8_b200 import quant

    path = Path(__file__).resolve().parents[1] / "examples" / "w8a8_block.py"
    spec = importlib.util.spec_from_file_location("w8a8_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    block = example.W8A8Block(dim, hidden, dtype, seed=tokens)
    g = rng(tokens)
    x, a = (torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    norm = dict(post_weight=block.norms[0], pre_weight=block.norms[1], gate=block.gates[0], scale=block.scale)
    x1, q, s = quant.residual_norm_quantized(x, a, **norm)
    rows = quant.gemm_scaled(q, s, *block.gate_up, gated=True, out_dtype=dtype, quantize=True)
    y = quant.linear(rows, *block.down)

    want_x, err_x, h, err_h = forward_ref(x, a, **norm, eps=1e-6, offset=0.0)
    close(x1, want_x, err_x, dtype)
    check_rows(q, s, h, err_h)
    hidden64, err = linear_ref(q, s, *block.gate_up, None, True)
    check_rows(rows.q, rows.scale, hidden64, err)
    check_close(y, *linear_ref(rows.q, rows.scale, *block.down, None, False), dtype)
