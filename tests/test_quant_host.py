"""8-bit operators, host side: the packed descriptors have the C compiler's
layout, and malformed arguments are refused before any device is touched."""

import struct
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
torch = pytest.importorskip("torch")

DESCS = {"rns8_cuda_quantize_desc": "QUANTIZE_DESC", "rns8_cuda_linear_desc": "LINEAR_DESC",
         "rns8_cuda_residual_norm_desc": "NORM_DESC", "rns8_cuda_residual_norm_backward_desc": "NORM_BACKWARD_DESC"}
INVALID, OVERFLOW_RISK = 1, 6
P = 4096  # an aligned address that is never read


@pytest.fixture(scope="module")
def quant():
    from rns8_b200 import quant

    return quant


def c_fields(name):
    """Field names of a descriptor in declaration order."""
    text = (ROOT / "include/rns8/rns8_quant.h").read_text()
    body = text.split(f"typedef struct {name} {{")[1].split("}")[0]
    out = []
    for line in body.splitlines():
        line = line.split("/*")[0].strip()
        if line.endswith(";"):
            out += [f.strip().lstrip("*") for f in line[:-1].split(",")]
            out[-len(line.split(",")):] = [f.split()[-1].lstrip("*") for f in out[-len(line.split(",")):]]
    return out


@pytest.mark.parametrize("name", DESCS)
def test_packed_descriptor_matches_c_layout(tmp_path, quant, name):
    fields = c_fields(name)
    src = tmp_path / "probe.c"
    probe = "".join(f'printf("%zu %zu\\n", offsetof({name}, {f}), sizeof((({name}*)0)->{f}));' for f in fields)
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "rns8/rns8_quant.h"\nint main(void){{'
                   f'printf("%zu\\n", sizeof({name}));{probe}return 0;}}')
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "probe")], check=True)
    lines = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.split("\n")
    packed = getattr(quant, DESCS[name])
    assert packed.size == int(lines[0])
    codes = []
    count = ""
    for ch in packed.format.lstrip("="):
        if ch.isdigit():
            count += ch
        else:
            codes += [ch] * int(count or 1)
            count = ""
    assert len(codes) == len(fields)
    at = 0
    for code, field, line in zip(codes, fields, lines[1:]):
        offset, size = map(int, line.split())
        assert (offset, size) == (at, struct.calcsize("=" + code)), field
        at += size


def linear_desc(quant, **change):
    f = dict(size=quant.LINEAR_DESC.size, abi=1, flags=0, device=0, a_type=3, out_type=0, reserved=0, m=4, n=8, k=16,
             ld_a=16, ld_w=16, ld_out=8, a=P, a_scale=P, w=P, w_scale=P, bias=0, out=P, out_scale=0, scratch=0, scratch_bytes=0,
             status=P, stream=0)
    f.update(change)
    return quant.LINEAR_DESC.pack(*f.values())


@pytest.mark.parametrize("change,want", [
    (dict(size=8), INVALID), (dict(abi=2), INVALID), (dict(flags=2), INVALID), (dict(reserved=1), INVALID),
    (dict(a_type=4), INVALID), (dict(out_type=3), INVALID), (dict(out_type=4), INVALID),
    (dict(out_scale=P), INVALID), (dict(out_type=3, out_scale=P + 2), INVALID), (dict(m=-1), INVALID), (dict(n=0), INVALID),
    (dict(k=0), INVALID), (dict(ld_a=15), INVALID), (dict(ld_w=15), INVALID), (dict(ld_out=7), INVALID),
    (dict(a=0), INVALID), (dict(w=0), INVALID), (dict(out=0), INVALID), (dict(w_scale=0), INVALID),
    (dict(a_scale=0), INVALID), (dict(a_type=0), INVALID), (dict(status=0), INVALID), (dict(status=P + 2), INVALID),
    (dict(a_type=0, a_scale=0, a=P + 1), INVALID), (dict(out=P + 1), INVALID), (dict(out_type=2, out=P + 2), INVALID),
    (dict(bias=P + 1), INVALID), (dict(ld_a=2**62), INVALID), (dict(m=2**31), INVALID),
    (dict(k=131072, ld_a=131072, ld_w=131072), OVERFLOW_RISK)])
def test_linear_refusals(quant, rns8, change, want):
    assert rns8.lib().rns8_cuda_linear_device(linear_desc(quant, **change)) == want
    if "status" not in change:  # the scratch query does not look at the status word
        assert rns8.lib().rns8_cuda_linear_scratch_bytes(linear_desc(quant, **change)) == 0


def test_linear_no_rows_is_a_no_op(quant, rns8):
    assert rns8.lib().rns8_cuda_linear_device(linear_desc(quant, m=0, a=0, out=0, a_scale=0)) == 0


@pytest.mark.parametrize("change", [dict(flags=1), dict(x_type=3), dict(rows=-1), dict(cols=0), dict(ld_x=9), dict(ld_q=9),
                                    dict(x=0), dict(q=0), dict(scale=0), dict(x=P + 1), dict(scale=P + 2)])
def test_quantize_refusals(quant, rns8, change):
    f = dict(size=quant.QUANTIZE_DESC.size, abi=1, flags=0, device=0, x_type=0, rows=2, cols=10, ld_x=10, ld_q=10, x=P,
             q=P, scale=P, stream=0)
    f.update(change)
    assert rns8.lib().rns8_cuda_quantize_rows_device(quant.QUANTIZE_DESC.pack(*f.values())) == INVALID


def norm_fields(quant, **change):
    f = dict(size=quant.NORM_DESC.size, abi=1, flags=0, device=0, type=0, weight_type=0, scale=1.0, eps=1e-6, offset=0.0,
             tokens=6, dim=10, groups=3, ld_x=10, ld_y=10, ld_gate=10, ld_x_out=10, ld_h=10, ld_q=10, x=P, y=P, post=P,
             pre=P, gate=P, x_out=P, h=P, q=0, q_scale=0, stream=0)
    f.update(change)
    return quant.NORM_DESC.pack(*f.values())


@pytest.mark.parametrize("change", [
    dict(flags=1), dict(type=3), dict(weight_type=1), dict(tokens=-1), dict(dim=0), dict(dim=32769, ld_x=40000, ld_y=40000,
                                                                                       ld_gate=40000, ld_x_out=40000,
                                                                                       ld_h=40000),
    dict(groups=4), dict(groups=0), dict(eps=-1.0), dict(eps=float("nan")), dict(ld_x=9), dict(ld_y=9), dict(ld_gate=9),
    dict(ld_x_out=9), dict(ld_h=9), dict(x=0), dict(y=0), dict(x_out=0), dict(pre=0), dict(h=0), dict(q=P, q_scale=0),
    dict(q=P, q_scale=P, ld_q=9), dict(x=P + 1), dict(post=P + 1), dict(pre=P + 1), dict(gate=P + 1)])
def test_norm_refusals(quant, rns8, change):
    assert rns8.lib().rns8_cuda_residual_norm_device(norm_fields(quant, **change)) == INVALID


@pytest.mark.parametrize("change", [
    dict(flags=1), dict(type=3), dict(groups=4), dict(ld_d_gate=9), dict(ld_d_x=9), dict(ld_d_y=9), dict(x_out=0),
    dict(y=0), dict(d_x=0), dict(d_y=0), dict(post=0), dict(pre=0), dict(gate=0), dict(d_post=P + 1), dict(d_gate=P + 2),
    dict(ld_dxo=9), dict(ld_dh=9)])
def test_norm_backward_refusals(quant, rns8, change):
    f = dict(size=quant.NORM_BACKWARD_DESC.size, abi=1, flags=0, device=0, type=0, weight_type=2, scale=1.0, eps=1e-6,
             offset=0.0, tokens=6, dim=10, groups=3, ld_dxo=10, ld_dh=10, ld_x_out=10, ld_y=10, ld_gate=10, ld_d_x=10,
             ld_d_y=10, ld_d_gate=10, dxo=P, dh=P, x_out=P, y=P, post=P, pre=P, gate=P, d_x=P, d_y=P, d_post=P, d_pre=P,
             d_gate=P, scratch=0, scratch_bytes=0, stream=0)
    f.update(change)
    packed = quant.NORM_BACKWARD_DESC.pack(*f.values())
    assert rns8.lib().rns8_cuda_residual_norm_backward_device(packed) == INVALID
    assert rns8.lib().rns8_cuda_residual_norm_backward_scratch_bytes(packed) == 0


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
