"""What the 8-bit operators do under autograd: the one with derivatives gives
them or says that it cannot, the others never drop one silently."""

import pytest

from test_gpu_quant_linear import operands, rng
from test_gpu_residual_norm import EPS32, backward_ref, close, make

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
fwAD = pytest.importorskip("torch.autograd.forward_ad")


@pytest.fixture(scope="module")
def quant():
    from rns8_b200 import quant

    return quant


@pytest.mark.parametrize("name", ["x", "y", "post_weight", "pre_weight", "gate"])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_residual_norm_refuses_forward_mode(quant, name, grad_mode):
    """A tangent was lost: the result was that of a constant."""
    t = make(4, 64, 2, torch.float32)
    with torch.set_grad_enabled(grad_mode), fwAD.dual_level():
        t[name] = fwAD.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(NotImplementedError):
            quant.residual_norm(**t)


def calls(quant, change):
    """Name -> the operator's results with one input changed by change."""
    a, s, w, ws, b = operands(4, 32, 64, 1)
    x = torch.randn(4, 64, generator=rng(2), device="cuda")
    t = make(4, 64, 2, torch.float32)
    g = [torch.randn(4, 64, generator=rng(3), device="cuda") for _ in range(2)]
    weights = {k: t[k] for k in ("post_weight", "pre_weight", "gate")}
    back = lambda **k: quant.residual_norm_backward(*g, t["x"], **{"y": t["y"], **weights, **k})  # noqa: E731
    found = {
        "quantize_rows": lambda: quant.quantize_rows(change(x)),
        "linear x": lambda: quant.linear(change(x), w, ws, bias=b),
        "linear w_scale": lambda: quant.linear(x, w, change(ws)),
        "linear bias": lambda: quant.linear(x, w, ws, bias=change(b)),
        "linear to int8": lambda: quant.linear(change(x), w, ws, quantize=True)[:2],
        "gemm_scaled a_scale": lambda: quant.gemm_scaled(a, change(s), w, ws),
        "gemm_scaled bias, gated": lambda: quant.gemm_scaled(a, s, w, ws, bias=change(b), gated=True)[:2],
    }
    for k in t:
        found[f"residual_norm_quantized {k}"] = lambda k=k: quant.residual_norm_quantized(**{**t, k: change(t[k])})
    for k in ("y", "post_weight", "pre_weight", "gate"):
        found[f"residual_norm_backward {k}"] = lambda k=k: back(**{k: change(t[k])})
    found["residual_norm_backward d_h"] = lambda: quant.residual_norm_backward(g[0], change(g[1]), t["x"], t["y"], **weights)
    return found


def results(value):
    return [r for r in (value if isinstance(value, tuple) else (value,)) if r is not None]


def test_a_gradient_through_the_others_raises(quant):
    """The values are those without autograd; asking for a gradient through
    them is an error, where before the results were constants."""
    plain, marked = calls(quant, lambda v: v), calls(quant, lambda v: v.clone().requires_grad_())
    for name in plain:
        want, got = results(plain[name]()), results(marked[name]())
        floats = [r for r in got if r.is_floating_point()]
        assert floats and all(r.requires_grad for r in floats), name
        for a, b in zip(got, want):
            assert torch.equal(a, b), name
        assert not any(r.requires_grad for r in want), name
        for r in floats:
            with pytest.raises(RuntimeError, match="not implemented"):
                r.sum().backward()
        with torch.no_grad():
            assert not any(r.requires_grad for r in results(marked[name]())), name


def test_the_others_refuse_forward_mode(quant):
    for name in calls(quant, lambda v: v):
        with fwAD.dual_level():
            call = calls(quant, lambda v: fwAD.make_dual(v, torch.ones_like(v)))[name]
            with pytest.raises(NotImplementedError):
                call()


def test_a_chain_of_products_carries_it(quant):
    """Through int8 rows the scales carry the mark."""
    _, _, w, ws, _ = operands(1, 64, 64, 1)
    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    y = quant.linear(quant.linear(x, w, ws, quantize=True), w, ws)
    assert y.requires_grad
    with pytest.raises(RuntimeError, match="not implemented"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,dim", [(1, 64), (5, 1001), (1300, 520), (1300, 515), (3, 8200)])
def test_a_32_bit_gate_has_a_32_bit_gradient(quant, tokens, dim, dtype):
    """With a row a token too, and for one token: it was rounded to the
    activations' 16 bits, so its precision depended on the batch."""
    t = make(tokens, dim, tokens, dtype, torch.float32)
    g = rng(dim)
    dxo, dh = (torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    args = {k: t[k] for k in ("y", "post_weight", "pre_weight", "gate")}
    got = quant.residual_norm_backward(dxo, dh, t["x"], **args, scale=0.7, eps=1e-5)
    value, terms = backward_ref(dxo, dh, t["x"], **args, scale=0.7, eps=1e-5, offset=0.0)[4]
    assert got[4].dtype == torch.float32
    close(got[4], value, 257 * EPS32 * terms, torch.float32)
    gate = t["gate"].clone().requires_grad_()
    xo, h = quant.residual_norm(**{**t, "gate": gate})
    torch.autograd.backward([xo, h], [dxo, dh])
    want = quant.residual_norm_backward(dxo, dh, xo.detach(), t["y"], post_weight=t["post_weight"],
                                        pre_weight=t["pre_weight"], gate=t["gate"])[4]
    assert torch.equal(gate.grad, want)
