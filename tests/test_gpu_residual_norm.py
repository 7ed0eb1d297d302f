"""residual_norm forward, its int8 form and its backward pass against the
formulas in 64 bits.

Error model (u32 = 2^-24): a row's sum of squares is a tree of at most 64
additions deep, so a row factor is within 48 u32; products add a few u32 more.
Every check allows 64 u32 (forward) or 256 u32 (backward) of the sum of the
magnitudes of the terms, sums over T tokens another T u32, plus one rounding
to the output type."""

import numpy as np
import pytest

from test_gpu_quant_linear import DTYPES, TINY, U, rng

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EPS32 = 2.0**-24


@pytest.fixture(scope="module")
def quant():
    from rns8_b200 import quant

    return quant


def make(tokens, dim, groups, dtype, wdtype=None, seed=0, post=True, pre=True, gate=True):
    g = rng(tokens * 31 + dim + seed)
    wdtype = wdtype or dtype
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = dict(x=(r(tokens, dim) * 2).to(dtype), y=(r(tokens, dim) * 3).to(dtype))
    t["post_weight"] = (1 + 0.3 * r(dim)).to(wdtype) if post else None
    t["pre_weight"] = (1 + 0.3 * r(dim)).to(wdtype) if pre else None
    t["gate"] = (0.5 + 0.5 * r(groups, dim)).to(wdtype) if gate else None
    return t


def d64(t):
    return None if t is None else t.double()


def forward_ref(x, y, post_weight, pre_weight, gate, scale, eps, offset):
    """x_out, h and bounds on the error of their 32-bit computation."""
    x, y, post, pre, gate = map(d64, (x, y, post_weight, pre_weight, gate))
    p = y
    if post is not None:
        p = y / torch.sqrt(y.square().mean(1, keepdim=True) + eps) * (offset + post)
    if gate is not None:
        p = p * gate.repeat_interleave(x.shape[0] // gate.shape[0], 0)
    xo = x + scale * p
    # offset + weight may cancel; its rounding is relative to its terms.
    loud = 1.0 if post is None else ((abs(offset) + post.abs()) / (offset + post).abs().clamp_min(1e-30)).clamp_max(1e6)
    err = 64 * EPS32 * (x.abs() + (scale * p).abs() * loud)
    if pre is None:
        return xo, err, None, None
    rho = 1 / torch.sqrt(xo.square().mean(1, keepdim=True) + eps)
    h = xo * rho * (offset + pre)
    rel = 64 * EPS32 + err.norm(dim=1, keepdim=True) / xo.norm(dim=1, keepdim=True).clamp_min(1e-30)
    herr = rho * (abs(offset) + pre.abs()) * (err + xo.abs() * rel)
    return xo, err, h, herr


def close(got, want, err, dtype):
    d = (got.double() - want).abs()
    tol = err * 1.01 + want.abs() * U[dtype] * 1.01 + TINY[dtype]
    assert not torch.isnan(d).any()
    assert bool((d <= tol).all()), float((d / tol).max())


SHAPES = [(1, 1, 1), (2, 3, 1), (1, 4096, 1), (5, 7, 5), (6, 64, 3), (64, 1001, 1), (33, 256, 33), (12, 2048, 4),
          (300, 520, 1), (7, 8192, 7), (4, 8193, 2), (2, 16384, 1), (3, 32768, 3), (40, 5000, 8), (1000, 96, 10)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,groups", SHAPES)
def test_forward(quant, tokens, dim, groups, dtype):
    t = make(tokens, dim, groups, dtype)
    xo, h = quant.residual_norm(**t, scale=0.7, eps=1e-5)
    wx, ex, wh, eh = forward_ref(**t, scale=0.7, eps=1e-5, offset=0.0)
    close(xo, wx, ex, dtype)
    close(h, wh, eh, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dim", [77, 640])
def test_forward_options(quant, dtype, post, pre, gate, dim):
    wdtype = torch.float32 if dim == 640 else dtype
    t = make(9, dim, 3, dtype, wdtype, post=post, pre=pre, gate=gate)
    xo, h = quant.residual_norm(**t, scale=-1.5, eps=1e-3, weight_offset=1.0)
    wx, ex, wh, eh = forward_ref(**t, scale=-1.5, eps=1e-3, offset=1.0)
    close(xo, wx, ex, dtype)
    assert (h is None) == (not pre)
    if pre:
        close(h, wh, eh, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim", [(1, 1), (3, 33), (1, 4096), (50, 1000), (8, 8200), (300, 256), (2, 32768)])
def test_quantized_form(quant, tokens, dim, dtype):
    """x_out is the same as the float form's; q * scale is within half a step
    of the 64-bit h, and the scale is its largest magnitude / 127."""
    t = make(tokens, dim, 1, dtype)
    t["pre_weight"][0] = 0
    xo, h = quant.residual_norm(**t)
    xq, q, s = quant.residual_norm_quantized(**t)
    assert torch.equal(xo, xq)
    _, _, wh, eh = forward_ref(**t, scale=1.0, eps=1e-6, offset=0.0)
    top = wh.abs().amax(1)
    assert bool(((s.double() * 127 - top).abs() <= eh.amax(1) + 4 * EPS32 * top + 1e-37).all())
    step = s.double()[:, None]
    assert bool(((q.double() * step - wh).abs() <= step * (0.5 + 127 * 4 * EPS32) + eh + 1e-37).all())
    assert int(q.to(torch.int16).abs().max()) <= 127


def test_special_rows(quant):
    """Zero rows stay finite (eps), an infinity or NaN stays in its own row."""
    for dtype in DTYPES:
        for dim in (48, 1001):
            t = make(6, dim, 1, dtype)
            t["x"][0] = 0
            t["y"][0] = 0
            xo, h = quant.residual_norm(**t)
            xq, q, s = quant.residual_norm_quantized(**t)
            assert not xo[0].any() and not h[0].any() and not q[0].any() and float(s[0]) == 0
            clean = xo.clone(), h.clone(), q.clone(), s.clone()
            t["y"][2, dim // 2] = float("inf")
            t["x"][4, dim - 1] = float("nan")
            xo, h = quant.residual_norm(**t)
            xq, q, s = quant.residual_norm_quantized(**t)
            keep = [0, 1, 3, 5]
            for got, want in zip((xo, h, q, s), clean):
                assert torch.equal(got[keep], want[keep])
            assert torch.isnan(h[2]).any() and torch.isnan(h[4]).all()
            assert not torch.isfinite(s[[2, 4]]).any() and not q[[2, 4]].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off,pad", [(0, 8), (1, 2), (8, 8)])
def test_strided(quant, dtype, off, pad):
    dim = 200
    t = make(10, dim + off + pad, 5, dtype)
    t = {k: v[..., off:off + dim] for k, v in t.items()}
    t["post_weight"], t["pre_weight"] = t["post_weight"].contiguous(), t["pre_weight"].contiguous()
    dense = {k: v.contiguous() for k, v in t.items()}
    for a, b in zip(quant.residual_norm(**t), quant.residual_norm(**dense)):
        assert torch.allclose(a.float(), b.float(), rtol=2 * U[dtype], atol=1e-5)
    t3 = {k: (v.unflatten(0, (5, 2)) if k in "xy" else v) for k, v in dense.items()}
    for a, b in zip(quant.residual_norm(**t3), quant.residual_norm(**dense)):
        assert a.shape == (5, 2, dim) and torch.equal(a.view(10, dim), b)


def backward_ref(dxo, dh, x, y, post_weight, pre_weight, gate, scale, eps, offset):
    """Gradients and the sums of the magnitudes of their terms."""
    dxo, dh, x, y, post, pre, gate = map(d64, (dxo, dh, x, y, post_weight, pre_weight, gate))
    tokens, dim = x.shape
    zero = torch.zeros_like(x)
    dxo = zero if dxo is None else dxo
    dh = zero if dh is None or pre is None else dh
    w2 = offset + pre if pre is not None else torch.zeros(dim, dtype=torch.float64, device="cuda")
    w1 = offset + post if post is not None else torch.ones(dim, dtype=torch.float64, device="cuda")
    groups = gate.shape[0] if gate is not None else 1
    g = scale * (gate.repeat_interleave(tokens // groups, 0) if gate is not None else torch.ones_like(x))
    rho = 1 / torch.sqrt(x.square().mean(1, keepdim=True) + eps)
    n, t = x * rho, dh * w2
    dx = dxo + rho * (t - n * (t * n).mean(1, keepdim=True))
    adx = dxo.abs() + rho * (t.abs() + n.abs() * (t * n).abs().mean(1, keepdim=True))
    sigma = 1 / torch.sqrt(y.square().mean(1, keepdim=True) + eps) if post is not None else torch.ones_like(rho)
    u = y * sigma
    dp = g * dx
    v = dp * w1
    av = (g * w1).abs() * adx
    dy, ady = v, av
    if post is not None:
        dy = sigma * (v - u * (v * u).mean(1, keepdim=True))
        ady = sigma * (av + u.abs() * (av * u.abs()).mean(1, keepdim=True))
    sums = lambda a: a.view(groups, -1, dim).sum(1)  # noqa: E731
    return [(dx, adx), (dy, ady),
            ((u * dp).sum(0), (u.abs() * g.abs() * adx).sum(0)) if post is not None else None,
            ((dh * n).sum(0), (dh * n).abs().sum(0)) if pre is not None else None,
            (sums(scale * u * w1 * dx), sums((scale * u * w1).abs() * adx)) if gate is not None else None]


def check_backward(quant, t, dxo, dh, dtype, scale=0.7, eps=1e-5, offset=0.0):
    args = {k: t[k] for k in ("y", "post_weight", "pre_weight", "gate")}
    got = quant.residual_norm_backward(dxo, dh, t["x"], **args, scale=scale, eps=eps, weight_offset=offset)
    want = backward_ref(dxo, dh, t["x"], **args, scale=scale, eps=eps, offset=offset)
    tokens = t["x"].shape[0]
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a is None) == (b is None), i
        if a is None:
            continue
        assert a.dtype == (dtype if i < 2 or (i == 4 and t["gate"].shape[0] == tokens) else torch.float32)
        close(a, b[0], (256 + (tokens if i >= 2 else 0)) * EPS32 * b[1], a.dtype)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,groups", SHAPES + [(1000, 64, 500), (777, 136, 1), (2000, 2048, 2),
                                                           (3000, 64, 1500), (900, 4096, 300), (450, 130, 150)])
def test_backward(quant, tokens, dim, groups, dtype):
    t = make(tokens, dim, groups, dtype)
    g = rng(dim)
    dxo = torch.randn(tokens, dim, generator=g, device="cuda").to(dtype)
    dh = torch.randn(tokens, dim, generator=g, device="cuda").to(dtype)
    got = check_backward(quant, t, dxo, dh, dtype)
    again = check_backward(quant, t, dxo, dh, dtype)
    for a, b in zip(got, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("has", [(True, True), (True, False), (False, True)])
def test_backward_options(quant, post, pre, gate, has):
    for dtype, wdtype, dim in ((torch.float32, None, 75), (torch.bfloat16, torch.float32, 640)):
        t = make(12, dim, 4, dtype, wdtype, post=post, pre=pre, gate=gate)
        g = rng(3)
        dxo = torch.randn(12, dim, generator=g, device="cuda").to(dtype) if has[0] else None
        dh = torch.randn(12, dim, generator=g, device="cuda").to(dtype) if has[1] else None
        check_backward(quant, t, dxo, dh, dtype, scale=-0.3, offset=1.0)


def test_backward_strided(quant):
    dim = 130
    for off, pad in ((0, 6), (1, 0), (8, 6)):
        t = make(14, dim + off + pad, 2, torch.bfloat16)
        t = {k: v[..., off:off + dim] for k, v in t.items()}
        t["post_weight"], t["pre_weight"] = t["post_weight"].contiguous(), t["pre_weight"].contiguous()
        g = rng(off)
        both = torch.randn(14, 2, dim, generator=g, device="cuda").to(torch.bfloat16)
        check_backward(quant, t, both[:, 0], both[:, 1], torch.bfloat16)


def test_autograd_against_differences(quant):
    """Directional derivatives of a scalar of both results against central
    differences of the forward kernel itself. With step 2^-6 and about 400
    terms of size 1, rounding costs under 1e-2 and the truncated third-order
    term about as much; gradients here are of size 10."""
    tokens, dim, step = 6, 32, 2.0**-6
    t = {k: v.requires_grad_() for k, v in make(tokens, dim, 3, torch.float32).items()}
    g = rng(5)
    c1 = torch.randn(tokens, dim, generator=g, device="cuda")
    c2 = torch.randn(tokens, dim, generator=g, device="cuda")

    def value(v):
        xo, h = quant.residual_norm(**v, scale=0.7)
        return (xo.double() * c1).sum() + (h.double() * c2).sum()

    xo, h = quant.residual_norm(**t, scale=0.7)
    ((xo * c1).sum() + (h * c2).sum()).backward()
    with torch.no_grad():
        for name in t:
            way = torch.randn(t[name].shape, generator=g, device="cuda")
            slope = float((t[name].grad.double() * way).sum())
            plus = {k: (v + step * way if k == name else v).detach() for k, v in t.items()}
            minus = {k: (v - step * way if k == name else v).detach() for k, v in t.items()}
            fd = float(value(plus) - value(minus)) / (2 * step)
            assert abs(fd - slope) <= 0.05 + 0.01 * abs(slope), (name, fd, slope)


def test_autograd_types_and_missing_gradients(quant):
    t = {k: v.requires_grad_() for k, v in make(8, 64, 8, torch.bfloat16).items()}
    xo, h = quant.residual_norm(**t)
    h.float().sum().backward()
    for v in t.values():
        assert v.grad is not None and v.grad.dtype == v.dtype and v.grad.shape == v.shape
    t = make(8, 64, 1, torch.float32, pre=False)
    t["gate"] = t["gate"][0].clone().requires_grad_()
    xo, h = quant.residual_norm(**t)
    assert h is None
    xo.sum().backward()
    assert t["gate"].grad.shape == (64,)


def test_offsets_past_32_bits(quant):
    """Rows 1.2e9 elements apart."""
    ld, dim = 1_200_000_000, 264
    buf = torch.empty(2 * ld + dim, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(buf, (3, dim), (ld, 1))
    t = make(3, dim, 1, torch.bfloat16)
    far.copy_(t["y"])
    want = quant.residual_norm(**t)
    dxo = torch.randn(3, dim, generator=rng(1), device="cuda").to(torch.bfloat16)
    args = {k: t[k] for k in ("post_weight", "pre_weight", "gate")}
    back = quant.residual_norm_backward(dxo, dxo, t["x"], t["y"], **args)
    for a, b in zip(quant.residual_norm(**{**t, "y": far}), want):
        assert torch.equal(a, b)
    for a, b in zip(quant.residual_norm_backward(dxo, dxo, t["x"], far, **args), back):
        assert torch.equal(a, b)


def test_no_tokens(quant):
    t = make(4, 64, 1, torch.float32)
    t["x"], t["y"] = t["x"][:0], t["y"][:0]
    xo, h = quant.residual_norm(**t)
    assert xo.shape == h.shape == (0, 64)
    got = quant.residual_norm_backward(xo, h, xo, t["y"], **{k: t[k] for k in ("post_weight", "pre_weight", "gate")})
    assert got[0].shape == (0, 64) and not got[2].any() and not got[3].any() and not got[4].any()
    assert got[4].shape == (1, 64)


def test_other_stream(quant):
    t = make(100, 512, 1, torch.bfloat16)
    want = quant.residual_norm(**t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = quant.residual_norm(**t)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals(quant):
    t = make(6, 64, 3, torch.bfloat16)
    bad = [dict(gate=t["gate"][:, :63]), dict(gate=torch.cat([t["gate"], t["gate"][:1]])), dict(y=t["y"][:, :63]),
           dict(y=t["y"].float()), dict(post_weight=t["post_weight"][:63]), dict(y=t["y"].cpu()),
           dict(pre_weight=t["pre_weight"].cpu())]
    for change in bad:
        with pytest.raises(ValueError):
            quant.residual_norm(**{**t, **change})
    for change in (dict(post_weight=t["post_weight"].float()), dict(gate=t["gate"].half())):
        with pytest.raises(TypeError):
            quant.residual_norm(**{**t, **change})
    wide = torch.zeros(1, 32769, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        quant.residual_norm(wide, wide)
    from rns8_b200 import Error

    with pytest.raises(Error):
        quant.residual_norm(**t, eps=-1.0)
