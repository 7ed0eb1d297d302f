"""8-bit operators, host side: the descriptors have the C compiler's layout,
and malformed arguments are refused before any device is touched."""

import ctypes as C
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
torch = pytest.importorskip("torch")

DESCS = {"rns8_cuda_quantize_desc": "QuantizeDesc", "rns8_cuda_linear_desc": "LinearDesc",
         "rns8_cuda_residual_norm_desc": "ResidualNormDesc",
         "rns8_cuda_residual_norm_backward_desc": "ResidualNormBackwardDesc"}
INVALID, OVERFLOW_RISK = 1, 6
P = 4096  # an aligned address that is never read


@pytest.fixture(scope="module")
def quant():
    from rns8_b200 import quant

    return quant


@pytest.mark.parametrize("name", DESCS)
def test_descriptor_matches_c_layout(tmp_path, rns8, name):
    mirror = getattr(rns8.abi, DESCS[name])
    fields = [f for f, _ in mirror._fields_]
    src = tmp_path / "probe.c"
    probe = "".join(f'printf("%zu %zu\\n", offsetof({name}, {f}), sizeof((({name}*)0)->{f}));' for f in fields)
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "rns8/rns8_quant.h"\nint main(void){{'
                   f'printf("%zu\\n", sizeof({name}));{probe}return 0;}}')
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "probe")], check=True)
    lines = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.split("\n")
    assert C.sizeof(mirror) == int(lines[0])
    for f, line in zip(fields, lines[1:]):
        assert (getattr(mirror, f).offset, getattr(mirror, f).size) == tuple(map(int, line.split())), f


def descriptor(kind, rns8, base, change):
    f = {**base, **change}
    d = getattr(rns8.abi, kind)()
    for name, value in f.items():
        setattr(d, name, value)
    return C.byref(d)


def linear_desc(rns8, **change):
    base = dict(a_type=3, m=4, n=8, k=16, ld_a=16, ld_w=16, ld_out=8, a=P, a_scale=P, w=P, w_scale=P, out=P, status=P)
    return descriptor("LinearDesc", rns8, base, change)


@pytest.mark.parametrize("change,want", [
    (dict(struct_size=8), INVALID), (dict(abi_version=2), INVALID), (dict(flags=2), INVALID), (dict(reserved=1), INVALID),
    (dict(a_type=4), INVALID), (dict(out_type=3), INVALID), (dict(out_type=4), INVALID),
    (dict(out_scale=P), INVALID), (dict(out_type=3, out_scale=P + 2), INVALID), (dict(m=-1), INVALID), (dict(n=0), INVALID),
    (dict(k=0), INVALID), (dict(ld_a=15), INVALID), (dict(ld_w=15), INVALID), (dict(ld_out=7), INVALID),
    (dict(a=0), INVALID), (dict(w=0), INVALID), (dict(out=0), INVALID), (dict(w_scale=0), INVALID),
    (dict(a_scale=0), INVALID), (dict(a_type=0), INVALID), (dict(status=0), INVALID), (dict(status=P + 2), INVALID),
    (dict(a_type=0, a_scale=0, a=P + 1), INVALID), (dict(out=P + 1), INVALID), (dict(out_type=2, out=P + 2), INVALID),
    (dict(bias=P + 1), INVALID), (dict(ld_a=2**62), INVALID), (dict(m=2**31), INVALID),
    (dict(k=131072, ld_a=131072, ld_w=131072), OVERFLOW_RISK)])
def test_linear_refusals(rns8, change, want):
    assert rns8.lib().rns8_cuda_linear_device(linear_desc(rns8, **change)) == want
    if "status" not in change:  # the scratch query does not look at the status word
        assert rns8.lib().rns8_cuda_linear_scratch_bytes(linear_desc(rns8, **change)) == 0


def test_linear_no_rows_is_a_no_op(rns8):
    assert rns8.lib().rns8_cuda_linear_device(linear_desc(rns8, m=0, a=0, out=0, a_scale=0)) == 0


@pytest.mark.parametrize("change", [dict(flags=1), dict(x_type=3), dict(rows=-1), dict(cols=0), dict(ld_x=9), dict(ld_q=9),
                                    dict(x=0), dict(q=0), dict(scale=0), dict(x=P + 1), dict(scale=P + 2)])
def test_quantize_refusals(rns8, change):
    base = dict(rows=2, cols=10, ld_x=10, ld_q=10, x=P, q=P, scale=P)
    assert rns8.lib().rns8_cuda_quantize_rows_device(descriptor("QuantizeDesc", rns8, base, change)) == INVALID


def norm_desc(rns8, **change):
    base = dict(scale=1.0, eps=1e-6, tokens=6, dim=10, groups=3, ld_x=10, ld_y=10, ld_gate=10, ld_x_out=10, ld_h=10,
                ld_q=10, x=P, y=P, post_weight=P, pre_weight=P, gate=P, x_out=P, h=P)
    return descriptor("ResidualNormDesc", rns8, base, change)


@pytest.mark.parametrize("change", [
    dict(flags=1), dict(type=3), dict(weight_type=1), dict(tokens=-1), dict(dim=0), dict(dim=32769, ld_x=40000, ld_y=40000,
                                                                                       ld_gate=40000, ld_x_out=40000,
                                                                                       ld_h=40000),
    dict(groups=4), dict(groups=0), dict(eps=-1.0), dict(eps=float("nan")), dict(ld_x=9), dict(ld_y=9), dict(ld_gate=9),
    dict(ld_x_out=9), dict(ld_h=9), dict(x=0), dict(y=0), dict(x_out=0), dict(pre_weight=0), dict(h=0), dict(q=P, q_scale=0),
    dict(q=P, q_scale=P, ld_q=9), dict(x=P + 1), dict(post_weight=P + 1), dict(pre_weight=P + 1), dict(gate=P + 1)])
def test_norm_refusals(rns8, change):
    assert rns8.lib().rns8_cuda_residual_norm_device(norm_desc(rns8, **change)) == INVALID


@pytest.mark.parametrize("change", [
    dict(flags=1), dict(type=3), dict(groups=4), dict(ld_d_gate=9), dict(ld_d_x=9), dict(ld_d_y=9), dict(x_out=0),
    dict(y=0), dict(d_x=0), dict(d_y=0), dict(post_weight=0), dict(pre_weight=0), dict(gate=0), dict(d_post=P + 1), dict(d_gate=P + 2),
    dict(ld_d_x_out=9), dict(ld_d_h=9)])
def test_norm_backward_refusals(rns8, change):
    base = dict(weight_type=2, scale=1.0, eps=1e-6, tokens=6, dim=10, groups=3, ld_d_x_out=10, ld_d_h=10, ld_x_out=10,
                ld_y=10, ld_gate=10, ld_d_x=10, ld_d_y=10, ld_d_gate=10, d_x_out=P, d_h=P, x_out=P, y=P, post_weight=P,
                pre_weight=P, gate=P, d_x=P, d_y=P, d_post=P, d_pre=P, d_gate=P)
    packed = descriptor("ResidualNormBackwardDesc", rns8, base, change)
    assert rns8.lib().rns8_cuda_residual_norm_backward_device(packed) == INVALID
    assert rns8.lib().rns8_cuda_residual_norm_backward_scratch_bytes(packed) == 0

def test_norm_backward_gate_gradient_type(rns8):
    """32 bits on request, for a 32-bit gate; ld and address go by that type."""
    base = dict(weight_type=2, scale=1.0, eps=1e-6, tokens=6, dim=10, groups=6, ld_d_x_out=10, ld_x_out=10, ld_y=10,
                ld_gate=10, ld_d_x=10, ld_d_y=10, ld_d_gate=10, d_x_out=P, x_out=P, y=P, post_weight=P, gate=P, d_x=P,
                d_y=P, d_post=P, d_gate=P)

    def need(**change):
        return rns8.lib().rns8_cuda_residual_norm_backward_scratch_bytes(
            descriptor("ResidualNormBackwardDesc", rns8, base, change))

    assert need() > 0 and need(flags=2) > 0  # scratch for d_post: the descriptor is valid
    assert need(d_gate=P + 2) > 0 and need(flags=2, d_gate=P + 2) == 0
    assert need(flags=2, weight_type=0) == 0 and need(flags=3) == 0 and need(flags=4) == 0
    d = norm_desc(rns8, flags=2)
    assert rns8.lib().rns8_cuda_residual_norm_device(d) == INVALID


def test_null_descriptors(rns8):
    for name in ("quantize_rows", "linear", "residual_norm", "residual_norm_backward"):
        assert getattr(rns8.lib(), f"rns8_cuda_{name}_device")(None) == INVALID


def test_python_refuses_cpu_tensors(quant):
    with pytest.raises(ValueError):
        quant.quantize_rows(torch.zeros(2, 4))
    with pytest.raises(ValueError):
        quant.residual_norm(torch.zeros(2, 4), torch.zeros(2, 4))
    with pytest.raises(TypeError):
        quant.quantize_rows(torch.zeros(2, 4, dtype=torch.float64))
