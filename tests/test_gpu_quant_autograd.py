"""What the 8-bit operators do under autograd: the one with derivatives gives
them or says that it cannot, the others never drop one silently."""

import pytest

from test_gpu_quant_linear import operands, rng
from test_gpu_residual_norm import make

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
