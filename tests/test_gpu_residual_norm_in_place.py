"""residual_norm over its own inputs (x_out = x, h = y; d_x = d_x_out, d_y =
d_h), through the C entry points, for each way rows are read and written: equal
bit for bit to the results in memory of their own."""

import ctypes as C

import pytest

from test_gpu_quant_linear import DTYPES, rng
from test_gpu_residual_norm import make
from test_gpu_residual_norm_offsets import Place, descriptor

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

# One token a block, the ring, rows wider than a block's registers or the ring;
# with (0, 0) on 16-byte boundaries where the width allows it.
SHAPES = [(5, 96), (40, 1001), (300, 4096), (3000, 1024), (3000, 1001), (3000, 4100), (700, 8192), (3, 12288), (3, 12289),
          (2, 32768), (9001, 64)]
LAYOUTS = [(0, 0), (3, 2)]


def places(tokens, dim, dtype, layout, *values):
    return [Place(tokens, dim, dtype, *layout, v) for v in values]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim", SHAPES)
def test_forward(tokens, dim, dtype, layout):
    from rns8_b200 import abi

    t = make(tokens, dim, 1, dtype)
    blank = torch.zeros(tokens, dim, device="cuda")

    def run(in_place):
        x, y = places(tokens, dim, dtype, layout, t["x"], t["y"])
        xo, h = (x, y) if in_place else places(tokens, dim, dtype, layout, blank, blank)
        q, scale = Place(tokens, dim, torch.int8, 0, -dim % 16), torch.empty(tokens, device="cuda")
        d = descriptor(abi, "ResidualNormDesc", tokens, dim, 1, dtype, dtype)
        d.x, d.ld_x, d.y, d.ld_y, d.gate, d.ld_gate = x.ptr, x.ld, y.ptr, y.ld, t["gate"].data_ptr(), dim
        d.post_weight, d.pre_weight = t["post_weight"].data_ptr(), t["pre_weight"].data_ptr()
        d.x_out, d.ld_x_out, d.h, d.ld_h = xo.ptr, xo.ld, h.ptr, h.ld
        d.q, d.ld_q, d.q_scale = q.ptr, q.ld, scale.data_ptr()
        assert abi.lib().rns8_cuda_residual_norm_device(C.byref(d)) == 0
        for p in (x, y, xo, h, q):
            assert p.holds()
        return xo.view, h.view, q.view, scale

    for got, want in zip(run(True), run(False)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("tokens,dim", SHAPES)
def test_backward(tokens, dim, per_token, dtype, layout):
    from rns8_b200 import abi

    groups = tokens if per_token else 1
    t = make(tokens, dim, groups, dtype)
    g = rng(dim)
    grads = [torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2)]
    blank = torch.zeros(tokens, dim, device="cuda")

    def run(in_place):
        dxo, dh, x, y = places(tokens, dim, dtype, layout, *grads, t["x"], t["y"])
        dx, dy = (dxo, dh) if in_place else places(tokens, dim, dtype, layout, blank, blank)
        dpost, dpre = (torch.empty(dim, device="cuda") for _ in range(2))
        dgate = torch.empty(groups, dim, device="cuda", dtype=dtype if groups == tokens else torch.float32)
        d = descriptor(abi, "ResidualNormBackwardDesc", tokens, dim, groups, dtype, dtype)
        d.d_x_out, d.ld_d_x_out, d.d_h, d.ld_d_h, d.x_out, d.ld_x_out = dxo.ptr, dxo.ld, dh.ptr, dh.ld, x.ptr, x.ld
        d.y, d.ld_y, d.gate, d.ld_gate = y.ptr, y.ld, t["gate"].data_ptr(), dim
        d.post_weight, d.pre_weight = t["post_weight"].data_ptr(), t["pre_weight"].data_ptr()
        d.d_x, d.ld_d_x, d.d_y, d.ld_d_y = dx.ptr, dx.ld, dy.ptr, dy.ld
        d.d_post, d.d_pre, d.d_gate, d.ld_d_gate = dpost.data_ptr(), dpre.data_ptr(), dgate.data_ptr(), dim
        need = abi.lib().rns8_cuda_residual_norm_backward_scratch_bytes(C.byref(d))
        scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
        d.scratch, d.scratch_bytes = scratch.data_ptr(), need
        assert abi.lib().rns8_cuda_residual_norm_backward_device(C.byref(d)) == 0
        for p in (dxo, dh, dx, dy, x, y):
            assert p.holds()
        return dx.view, dy.view, dpost, dpre, dgate

    for got, want in zip(run(True), run(False)):
        assert torch.equal(got, want)
