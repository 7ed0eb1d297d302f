"""Broadcast operands (rows that share memory) of the 8-bit operators: as if
copied out, and gradients summed over what shares an element."""

import pytest

from test_gpu_quant_linear import DTYPES, operands, rng
from test_gpu_residual_norm import make

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def quant():
    from rns8_b200 import quant

    return quant


def same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 1001])
def test_broadcast_operands(quant, dim, dtype):
    g = rng(dim)
    one = torch.randn(1, dim, generator=g, device="cuda").to(dtype)
    many, dense = one.expand(6, dim), one.expand(6, dim).contiguous()
    windows = torch.randn(dim + 5, generator=g, device="cuda").to(dtype).unfold(0, dim, 1)
    assert windows.shape == (6, dim)
    _, _, w, ws, _ = operands(1, 40, dim, 1)
    ws = ws / 32
    for shared, own in ((many, dense), (windows, windows.contiguous())):
        same(quant.quantize_rows(shared), quant.quantize_rows(own))
        same([quant.linear(shared, w, ws)], [quant.linear(own, w, ws)])
        t = make(6, dim, 6, dtype)
        weights = {k: t[k] for k in ("post_weight", "pre_weight")}
        for x, y, gate in ((shared, t["y"], t["gate"]), (t["x"], shared, t["gate"]), (t["x"], t["y"], shared)):
            full = x.contiguous(), y.contiguous()
            same(quant.residual_norm(x, y, gate=gate, **weights),
                 quant.residual_norm(*full, gate=gate.contiguous(), **weights))
            same(quant.residual_norm_backward(shared, shared, x, y, gate=gate, **weights),
                 quant.residual_norm_backward(own, own, *full, gate=gate.contiguous(), **weights))
    row = w[:1].expand(40, dim)
    same([quant.linear(dense, row, ws)], [quant.linear(dense, row.contiguous(), ws)])


def test_gradients_of_broadcast_operands(quant):
    t = make(6, 64, 6, torch.float32)
    t["gate"], t["x"] = t["gate"][:1].clone(), t["x"][:1].clone()
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    spread = {k: v.expand(6, 64) if k in ("x", "gate") else v for k, v in leaves.items()}
    xo, h = quant.residual_norm(**spread)
    (xo.square().sum() + h.square().sum()).backward()
    dense = {k: v.detach().clone().requires_grad_() for k, v in {**t, "x": spread["x"], "gate": spread["gate"]}.items()}
    xo, h = quant.residual_norm(**dense)
    (xo.square().sum() + h.square().sum()).backward()
    for k in t:
        want = dense[k].grad.sum(0, keepdim=True) if k in ("x", "gate") else dense[k].grad
        assert torch.equal(leaves[k].grad, want), k
