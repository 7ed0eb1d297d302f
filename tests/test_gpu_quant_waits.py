"""Bounded waits of the 8-bit operators that run out. The limit is made a single
cycle: the norms then read every row from global memory and answer as ever; the
products, where data was late, set the status word and return, and what comes
after is as if nothing had happened. Waits for a kernel's own copies and
products before it leaves keep their full limit."""

import pytest

from test_gpu_quant_linear import DTYPES, operands, rng
from test_gpu_residual_norm import make

torch = pytest.importorskip("torch")


@pytest.fixture
def limit(rns8):
    """Sets the limit; the usual one afterwards."""

    def put(cycles):
        assert rns8.lib().rns8_cuda_quant_wait_limit(cycles) == 0

    yield put
    put(0)


def test_limit_refusals(rns8, limit):
    for bad in (4_000_000_001, 2**63, 2**64 - 1):
        assert rns8.lib().rns8_cuda_quant_wait_limit(bad) == 1
    limit(1)
    limit(4_000_000_000)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,groups", [(3000, 4096, 1), (2500, 8192, 10), (700, 16384, 1), (20000, 256, 1)])
def test_norm_forward(limit, tokens, dim, groups, dtype):
    from rns8_b200 import quant

    t = make(tokens, dim, groups, dtype)
    want = *quant.residual_norm(**t), *quant.residual_norm_quantized(**t)
    limit(1)
    for _ in range(2):
        for got, w in zip((*quant.residual_norm(**t), *quant.residual_norm_quantized(**t)), want):
            assert torch.equal(got, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,groups", [(3000, 4096, 1), (3000, 4096, 3000), (2500, 8192, 10), (4000, 264, 4000),
                                               (4001, 1001, 1), (4001, 1001, 4001)])
def test_norm_backward(limit, tokens, dim, groups, dtype):
    from rns8_b200 import quant

    t = make(tokens, dim, groups, dtype)
    args = {k: t[k] for k in ("y", "post_weight", "pre_weight", "gate")}
    g = rng(dim)
    grads = [torch.randn(tokens, dim, generator=g, device="cuda").to(dtype) for _ in range(2)]
    want = quant.residual_norm_backward(*grads, t["x"], **args)
    limit(1)
    for _ in range(2):
        for got, w in zip(quant.residual_norm_backward(*grads, t["x"], **args), want):
            assert torch.equal(got, w)


# Tokens on lanes, several tiles a block; channels on lanes by one block and by a
# cluster, 16 and 128 tokens to a tile. The last two may find all their data there
# in time.
PRODUCTS = [(2500, 8200, 1104, False), (2500, 4100, 1104, True), (6536, 273, 64, False), (304, 201, 3952, True),
            (1, 201, 64, False), (5, 202, 1936, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,gated", PRODUCTS)
def test_product_reports(limit, m, n, k, gated):
    """A product under the short limit reports, or its result is right; so is
    the next one's under the usual limit."""
    from rns8_b200 import quant

    a, s, w, ws, b = operands(m, 2 * n if gated else n, k, m + n)
    s = s / k**0.5

    def run():
        return quant.gemm_scaled(a, s, w, ws, bias=b, gated=gated, quantize=False)

    want = run()
    quant.check_status(0)
    limit(1)
    got = run()
    try:
        quant.check_status(0)
        assert torch.equal(got, want) and m < 10
    except RuntimeError as e:
        assert "0x100" in str(e)
    limit(0)
    assert torch.equal(run(), want)
    quant.check_status(0)
