"""residual_norm with several tokens a block: rows through a shared-memory ring
that is filled again and wraps, sums whose slots alternate, int8 rows token
after token. Formulas and error model are those of test_gpu_residual_norm."""

import ctypes as C

import pytest

from test_gpu_quant_linear import DTYPES, rng
from test_gpu_residual_norm import EPS32, check_backward, close, forward_ref, make
from test_gpu_residual_norm_offsets import Place, descriptor

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def quant():
    from rns8_b200 import quant

    return quant


# Blocks of 8 warps and more with one to three rows in the ring, of one warp (no
# barrier in its sums), rows as wide as the ring takes, and a last round that
# leaves some blocks without a token.
SHAPES = [(3000, 4096, 1), (3000, 4096, 3000), (2500, 8192, 10), (700, 16384, 7), (20000, 256, 1), (9001, 64, 1),
          (4000, 1032, 4000), (1777, 2056, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,groups", SHAPES)
def test_forward(quant, tokens, dim, groups, dtype):
    t = make(tokens, dim, groups, dtype)
    wx, ex, wh, eh = forward_ref(**t, scale=0.7, eps=1e-5, offset=0.0)
    xo, h = quant.residual_norm(**t, scale=0.7, eps=1e-5)
    close(xo, wx, ex, dtype)
    close(h, wh, eh, dtype)
    xq, q, s = quant.residual_norm_quantized(**t, scale=0.7, eps=1e-5)
    assert torch.equal(xq, xo)
    check_rows(q, s, wh, eh)


def check_rows(q, s, wh, eh):
    top, step = wh.abs().amax(1), s.double()[:, None]
    assert bool(((s.double() * 127 - top).abs() <= eh.amax(1) + 4 * EPS32 * top + 1e-37).all())
    assert bool(((q.double() * step - wh).abs() <= step * (0.5 + 127 * 4 * EPS32) + eh + 1e-37).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("tokens,dim", [(3000, 1024), (9001, 64)])
def test_forward_options(quant, tokens, dim, post, pre, gate, dtype):
    t = make(tokens, dim, tokens // 1000 if tokens % 1000 == 0 else 1, dtype, torch.float32, post=post, pre=pre, gate=gate)
    wx, ex, wh, eh = forward_ref(**t, scale=-1.5, eps=1e-3, offset=1.0)
    xo, h = quant.residual_norm(**t, scale=-1.5, eps=1e-3, weight_offset=1.0)
    close(xo, wx, ex, dtype)
    assert (h is None) == (not pre)
    if pre:
        close(h, wh, eh, dtype)
        _, q, s = quant.residual_norm_quantized(**t, scale=-1.5, eps=1e-3, weight_offset=1.0)
        check_rows(q, s, wh, eh)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim", [(3000, 4096), (9001, 64)])
def test_both_results_at_once(tokens, dim, dtype):
    """Floats and int8 rows from one call, with guards around each row."""
    from rns8_b200 import abi, quant

    t = make(tokens, dim, 1, dtype)
    xo, h = (Place(tokens, dim, dtype, 0, 8) for _ in range(2))
    q, scale = Place(tokens, dim, torch.int8, 0, 8), torch.empty(tokens, device="cuda")
    d = descriptor(abi, "ResidualNormDesc", tokens, dim, 1, dtype, dtype)
    d.x, d.ld_x, d.y, d.ld_y, d.gate, d.ld_gate = t["x"].data_ptr(), dim, t["y"].data_ptr(), dim, t["gate"].data_ptr(), dim
    d.post_weight, d.pre_weight = t["post_weight"].data_ptr(), t["pre_weight"].data_ptr()
    d.x_out, d.ld_x_out, d.h, d.ld_h, d.q, d.ld_q, d.q_scale = xo.ptr, xo.ld, h.ptr, h.ld, q.ptr, q.ld, scale.data_ptr()
    assert abi.lib().rns8_cuda_residual_norm_device(C.byref(d)) == 0
    args = dict(scale=0.7, eps=1e-5, weight_offset=0.5)
    want_x, want_h = quant.residual_norm(**t, **args)
    _, want_q, want_s = quant.residual_norm_quantized(**t, **args)
    for got, want in ((xo.view, want_x), (h.view, want_h), (q.view, want_q), (scale, want_s)):
        assert torch.equal(got, want)
    assert xo.holds() and h.holds() and q.holds()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim", [(3000, 4096), (20000, 256), (3000, 1001)])
def test_special_rows_stay_apart(quant, tokens, dim, dtype):
    """Zeros, an infinity or a NaN in some tokens leave every other token's bits."""
    t = make(tokens, dim, 1, dtype)
    clean = *quant.residual_norm(**t), *quant.residual_norm_quantized(**t)[1:]
    at = torch.tensor([0, 1, 147, 148, 149, 600, 1183, 1184, tokens - 1], device="cuda")
    t["x"][at] = 0
    t["y"][at] = 0
    t["y"][at[1::3], dim // 2] = float("inf")
    t["x"][at[2::3], dim - 1] = float("nan")
    got = *quant.residual_norm(**t), *quant.residual_norm_quantized(**t)[1:]
    rest = torch.ones(tokens, dtype=torch.bool, device="cuda")
    rest[at] = False
    for a, b in zip(got, clean):
        assert torch.equal(a[rest], b[rest])
    xo, h, q, s = got
    zero = at[0::3]
    assert not xo[zero].any() and not h[zero].any() and not q[zero].any() and not s[zero].any()
    bad = torch.cat([at[1::3], at[2::3]])
    assert not torch.isfinite(s[bad]).any() and not q[bad].any() and torch.isnan(h[bad]).any(1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,groups", [(3000, 4096, 1), (3000, 4096, 3000), (2500, 8192, 10), (9001, 64, 1),
                                               (9000, 264, 9000), (4001, 1001, 1)])
def test_backward(quant, tokens, dim, groups, dtype):
    t = make(tokens, dim, groups, dtype)
    g = rng(dim)
    dxo, dh = (torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    got = check_backward(quant, t, dxo, dh, dtype)
    for a, b in zip(check_backward(quant, t, dxo, dh, dtype), got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("tokens,dim", [(148, 4096), (149, 4096), (290, 4096), (290, 4095), (440, 2056), (440, 2559),
                                        (443, 2048), (296, 3080)])
def test_backward_around_one_token_a_block(quant, tokens, dim, per_token, dtype):
    """Either side of the choice between rows in registers and the ring."""
    t = make(tokens, dim, tokens if per_token else 1, dtype)
    g = rng(dim)
    dxo, dh = (torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    check_backward(quant, t, dxo, dh, dtype)
