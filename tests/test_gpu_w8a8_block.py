"""The 8-bit operators together: the example block against 32-bit floats, and
its command."""

import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "w8a8_block.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("w8a8_block", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("tokens,dim,hidden", [(1, 256, 512), (5, 512, 320), (64, 1024, 2048), (300, 520, 1000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block_against_floats(example, tokens, dim, hidden, dtype):
    """Rounding Gaussian rows to 255 levels of their largest magnitude (4 to 5
    standard deviations) costs about 1 % of a row's norm; three quantised
    operands and a norm keep the update within a few per cent, and the update
    is about half of the residual."""
    block = example.W8A8Block(dim, hidden, dtype, seed=tokens)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x, a = (torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    for got, want in zip(block.forward(x, a), block.reference(x, a)):
        assert got.dtype == dtype and example.relative_error(got, want) < 0.03


def test_command():
    out = subprocess.run([sys.executable, str(EXAMPLE), "--tokens", "9", "--dim", "512", "--hidden", "1024", "--steps", "3"],
                         capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert "us a block" in out.stdout and "relative error" in out.stdout
