"""Gradients of residual_norm at the ends of its range: rows far larger or
smaller than 1, eps of zero or near it, rows of zeros, infinities where a value
takes no part, offsets without a weight. Formulas and error model are those of
test_gpu_residual_norm; rows of each kernel form are among the shapes."""

import pytest

from test_gpu_quant_linear import rng
from test_gpu_residual_norm import check_backward, make

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def quant():
    from rns8_b200 import quant

    return quant


# (tokens, dim, groups): one row a block, aligned and not; the ring, aligned
# and not, with shared gate rows and a row a token; wider than the ring's rows.
FORMS = [(5, 96, 1), (5, 1001, 5), (1500, 256, 3), (1400, 1001, 1), (1300, 520, 1300), (1300, 515, 1300),
         (3, 8200, 1), (2, 8199, 2)]


def gradients(tokens, dim, dtype, seed=0):
    g = rng(dim + seed)
    return [torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rms,eps", [(1e16, 1e-6), (1e14, 1e-6), (1e-13, 0.0), (1e-15, 0.0), (1e-17, 0.0)])
@pytest.mark.parametrize("tokens,dim,groups", FORMS)
def test_row_magnitudes(quant, tokens, dim, groups, rms, eps, dtype):
    """The powers of 1/rms that the gradients hold are never formed by
    themselves: the cube of 1e-14 or of 1e13 is outside the 32-bit range."""
    for of in ("x", "y", "xy"):
        t = make(tokens, dim, groups, dtype)
        for k in of:
            t[k] = (t[k].float() * (rms / 2)).to(dtype)
        dxo, dh = gradients(tokens, dim, dtype)
        check_backward(quant, t, dxo, dh, dtype, eps=eps)
        check_backward(quant, t, None, dh, dtype, eps=eps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,dim,groups", FORMS)
def test_zero_rows_and_a_tiny_eps(quant, tokens, dim, groups, dtype):
    t = make(tokens, dim, groups, dtype)
    t["x"][0] = 0
    t["y"][tokens // 2] = 0
    dxo, dh = gradients(tokens, dim, dtype)
    check_backward(quant, t, dxo, dh, dtype, eps=1e-30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,dim,groups", FORMS)
def test_without_pre_weight_x_out_takes_no_part(quant, tokens, dim, groups, dtype):
    """d_x is d_x_out then, whatever x_out holds."""
    for post in (True, False):
        t = make(tokens, dim, groups, dtype, pre=False, post=post)
        dxo, _ = gradients(tokens, dim, dtype)
        args = {k: t[k] for k in ("post_weight", "gate")}
        want = quant.residual_norm_backward(dxo, None, t["x"], t["y"], **args)
        assert torch.equal(want[0], dxo)
        x = t["x"].clone()
        x[0, dim // 2], x[1, 0], x[tokens - 1, dim - 1] = float("inf"), float("nan"), float("-inf")
        for a, b in zip(quant.residual_norm_backward(dxo, None, x, t["y"], **args), want):
            assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,dim,groups", FORMS)
def test_without_post_weight_y_enters_the_gates_gradient_alone(quant, tokens, dim, groups, dtype):
    dxo, dh = gradients(tokens, dim, dtype)
    bad = [(0, dim // 2, float("inf")), (1, 0, float("nan")), (tokens - 1, dim - 1, float("-inf"))]
    for gate in (True, False):
        t = make(tokens, dim, groups, dtype, post=False, gate=gate)
        args = {k: t[k] for k in ("pre_weight", "gate")}
        want = quant.residual_norm_backward(dxo, dh, t["x"], t["y"], **args)
        y = t["y"].clone()
        for row, col, value in bad:
            y[row, col] = value
        got = quant.residual_norm_backward(dxo, dh, t["x"], y, **args)
        for i in (0, 1, 3):
            assert torch.equal(got[i], want[i]), i
        if gate:
            of = torch.zeros_like(want[4], dtype=torch.bool)
            for row, col, _ in bad:
                of[row // (tokens // groups), col] = True
            assert not torch.isfinite(got[4][of]).any() and torch.equal(got[4][~of], want[4][~of])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [3e8, -1e30, 1e30])
@pytest.mark.parametrize("tokens,dim,groups", FORMS)
def test_offset_belongs_to_a_weight(quant, tokens, dim, groups, offset, dtype):
    """An absent weight is a factor of 1 whatever the offset."""
    t = make(tokens, dim, groups, dtype, post=False, pre=False)
    dxo, _ = gradients(tokens, dim, dtype)
    for gate in (t["gate"], None):
        want = quant.residual_norm_backward(dxo, None, t["x"], t["y"], gate=gate)
        got = quant.residual_norm_backward(dxo, None, t["x"], t["y"], gate=gate, weight_offset=offset)
        for a, b in zip(got, want):
            assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,dim,groups", FORMS)
def test_bad_rows_stay_apart(quant, tokens, dim, groups, dtype):
    """An infinity or NaN makes its own token's gradients NaN, as the formulas
    do, and leaves every other token's bits."""
    t = make(tokens, dim, groups, dtype)
    args = {k: t[k] for k in ("post_weight", "pre_weight", "gate")}
    dxo, dh = gradients(tokens, dim, dtype)
    want = quant.residual_norm_backward(dxo, dh, t["x"], t["y"], **args)
    for of in range(4):
        rows = [v.clone() for v in (dxo, dh, t["x"], t["y"])]
        rows[of][0, dim // 3], rows[of][tokens - 1, dim - 1] = float("nan"), float("inf")
        got = quant.residual_norm_backward(*rows, **args)
        for a, b in zip(got[:2], want[:2]):
            assert torch.equal(a[1:tokens - 1], b[1:tokens - 1])
        assert not torch.isfinite(got[1][[0, tokens - 1]]).any()  # d_y depends on all of its token
        if of == 3:  # y reaches d_y and the gate, not d_x
            assert torch.equal(got[0], want[0])
        else:
            assert not torch.isfinite(got[0][[0, tokens - 1]]).all(1).any()
