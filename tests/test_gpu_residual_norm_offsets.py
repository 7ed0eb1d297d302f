"""Residual norms of rows that start anywhere: odd widths, every tensor at its
own offset and pitch, few and many tokens, with guard elements around every
output row. Formulas and error model are those of test_gpu_residual_norm."""

import ctypes as C

import pytest

from test_gpu_quant_linear import DTYPES, rng
from test_gpu_residual_norm import EPS32, backward_ref, close, forward_ref, make

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

GUARD = 77.0


class Place:
    """Puts rows (or a vector) `off` elements into a buffer of guard values,
    `pad` elements between them; holds reports whether the guards still stand."""

    def __init__(self, rows, dim, dtype, off, pad, value=None):
        self.rows, self.dim, self.off, self.ld = rows, dim, off, dim + pad
        self.buf = torch.full((off + rows * self.ld + 16,), GUARD, device="cuda").to(dtype)
        self.view = torch.as_strided(self.buf, (rows, dim), (self.ld, 1), off)
        if value is not None:
            self.view.copy_(value.view(rows, dim))

    def holds(self):
        left = self.buf.clone()
        torch.as_strided(left, (self.rows, self.dim), (self.ld, 1), self.off).fill_(GUARD)
        return bool((left == GUARD).all())

    @property
    def ptr(self):
        return self.view.data_ptr()


def code(dtype):
    return {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}[dtype]


SHAPES = [(1, 1), (1, 1001), (3, 9), (5, 264), (40, 2050), (700, 5), (700, 257), (650, 1001), (600, 2056), (601, 4099),
          (600, 8191), (5, 8199)]
# Offsets and pitches of the tensors in order: all different, or all the same.
LAYOUTS = [[(1, 0), (2, 3), (3, 1), (0, 2), (5, 5), (6, 0), (7, 4), (4, 1), (3, 0)], [(0, 0)] * 9]


def descriptor(abi, kind, tokens, dim, groups, dtype, wdtype):
    d = getattr(abi, kind)()
    d.tokens, d.dim, d.groups, d.type, d.weight_type = tokens, dim, groups, code(dtype), code(wdtype)
    d.scale, d.eps, d.weight_offset = 0.7, 1e-5, 0.5
    d.stream = torch.cuda.current_stream().cuda_stream
    return d


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype,wdtype", [(t, t) for t in DTYPES] + [(torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("tokens,dim", SHAPES + [(600, 12289)])
def test_forward(tokens, dim, dtype, wdtype, layout):
    from rns8_b200 import abi

    groups = 5 if tokens % 5 == 0 else 1
    t = make(tokens, dim, groups, dtype, wdtype)
    (x, y, gate, post, pre) = (Place(r, dim, k, *at, v) for r, k, at, v in (
        (tokens, dtype, layout[0], t["x"]), (tokens, dtype, layout[1], t["y"]), (groups, wdtype, layout[2], t["gate"]),
        (1, wdtype, layout[3], t["post_weight"]), (1, wdtype, layout[4], t["pre_weight"])))
    xo, h = Place(tokens, dim, dtype, *layout[5]), Place(tokens, dim, dtype, *layout[6])
    q, scale = Place(tokens, dim, torch.int8, *layout[7]), torch.empty(tokens, device="cuda")
    d = descriptor(abi, "ResidualNormDesc", tokens, dim, groups, dtype, wdtype)
    d.x, d.ld_x, d.y, d.ld_y, d.gate, d.ld_gate = x.ptr, x.ld, y.ptr, y.ld, gate.ptr, gate.ld
    d.post_weight, d.pre_weight = post.ptr, pre.ptr
    d.x_out, d.ld_x_out, d.h, d.ld_h, d.q, d.ld_q, d.q_scale = xo.ptr, xo.ld, h.ptr, h.ld, q.ptr, q.ld, scale.data_ptr()
    assert abi.lib().rns8_cuda_residual_norm_device(C.byref(d)) == 0
    want_x, err_x, want_h, err_h = forward_ref(**t, scale=0.7, eps=1e-5, offset=0.5)
    close(xo.view, want_x, err_x, dtype)
    close(h.view, want_h, err_h, dtype)
    step = scale.double()[:, None]
    assert bool(((q.view.double() * step - want_h).abs() <= step * (0.5 + 127 * 4 * EPS32) + err_h + 1e-37).all())
    for p in (xo, h, q):
        assert p.holds()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype,wdtype", [(t, t) for t in DTYPES] + [(torch.float16, torch.float32)])
@pytest.mark.parametrize("rows_per_gate", [0, 1])
@pytest.mark.parametrize("tokens,dim", SHAPES)
def test_backward(tokens, dim, rows_per_gate, dtype, wdtype, layout):
    from rns8_b200 import abi

    groups = tokens if rows_per_gate else (5 if tokens % 5 == 0 else 1)
    t = make(tokens, dim, groups, dtype, wdtype)
    g = rng(dim)
    grads = [torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2)]
    dxo, dh = Place(tokens, dim, dtype, *layout[0], grads[0]), Place(tokens, dim, dtype, *layout[1], grads[1])
    x, y = Place(tokens, dim, dtype, *layout[2], t["x"]), Place(tokens, dim, dtype, *layout[3], t["y"])
    gate, post = Place(groups, dim, wdtype, *layout[4], t["gate"]), Place(1, dim, wdtype, *layout[5], t["post_weight"])
    pre = Place(1, dim, wdtype, *layout[6], t["pre_weight"])
    dx, dy = Place(tokens, dim, dtype, *layout[7]), Place(tokens, dim, dtype, *layout[8])
    dpost, dpre = Place(1, dim, torch.float32, *layout[0]), Place(1, dim, torch.float32, *layout[1])
    dgate = Place(groups, dim, dtype if groups == tokens else torch.float32, *layout[2])
    d = descriptor(abi, "ResidualNormBackwardDesc", tokens, dim, groups, dtype, wdtype)
    d.d_x_out, d.ld_d_x_out, d.d_h, d.ld_d_h, d.x_out, d.ld_x_out = dxo.ptr, dxo.ld, dh.ptr, dh.ld, x.ptr, x.ld
    d.y, d.ld_y, d.gate, d.ld_gate, d.post_weight, d.pre_weight = y.ptr, y.ld, gate.ptr, gate.ld, post.ptr, pre.ptr
    d.d_x, d.ld_d_x, d.d_y, d.ld_d_y, d.d_post, d.d_pre = dx.ptr, dx.ld, dy.ptr, dy.ld, dpost.ptr, dpre.ptr
    d.d_gate, d.ld_d_gate = dgate.ptr, dgate.ld
    need = abi.lib().rns8_cuda_residual_norm_backward_scratch_bytes(C.byref(d))
    scratch = torch.full((need + 64,), 99, dtype=torch.uint8, device="cuda")
    d.scratch, d.scratch_bytes = scratch.data_ptr(), need
    assert abi.lib().rns8_cuda_residual_norm_backward_device(C.byref(d)) == 0
    want = backward_ref(*grads, t["x"], *(t[k] for k in ("y", "post_weight", "pre_weight", "gate")), scale=0.7, eps=1e-5,
                        offset=0.5)
    for i, (p, w) in enumerate(zip((dx, dy, dpost, dpre, dgate), want)):
        value, terms = (a.view(p.rows, dim) for a in w)
        close(p.view, value, (256 + (tokens if i >= 2 else 0)) * EPS32 * terms, p.buf.dtype)
        assert p.holds(), i
    assert bool((scratch[need:] == 99).all())
