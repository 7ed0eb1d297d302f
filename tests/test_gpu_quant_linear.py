"""quantize_rows, gemm_scaled and linear against plain 64-bit forms.

Quantisation is defined in 32-bit operations, so q and scale must equal the
same operations done in numpy. The product's sum is exact; what follows it is
a handful of 32-bit operations, each within 2^-24 relative, and one rounding
to the output type (unit roundoff 2^-8 bf16, 2^-11 f16, 2^-24 f32)."""

import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24, torch.float32: 2.0**-126}
DTYPES = list(U)


@pytest.fixture(scope="module")
def quant():
    from rns8_b200 import quant

    return quant


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def quantize_ref(x):
    """q and scale by the definition, in numpy's 32-bit operations."""
    x = x.float().cpu().numpy()
    a = np.abs(x).max(axis=1)  # NaN wins
    with np.errstate(all="ignore"):
        scale = np.where(np.isfinite(a), a / np.float32(127), a).astype(np.float32)
        inv = (np.float32(127) / a).astype(np.float32)
        zero = ~np.isfinite(a) | (a < np.float32(127 * 2.0**-126))
        scale[np.isfinite(a) & zero] = 0
        q = np.rint(x * np.where(zero, 0, inv)[:, None])
    q[zero] = 0
    return q.astype(np.int8), scale


def check_quantized(quant, x):
    q, s = quant.quantize_rows(x)
    wq, ws = quantize_ref(x)
    assert np.array_equal(q.cpu().numpy(), wq)
    assert np.array_equal(s.cpu().numpy(), ws, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 4096), (5, 8), (17, 1001), (130, 64), (2, 8192), (2, 8200),
                                       (3, 32768), (2, 32769), (2, 50001), (300, 257)])
def test_quantize_rows(quant, dtype, rows, cols):
    x = torch.randn(rows, cols, generator=rng(rows * cols), device="cuda").mul_(3).to(dtype)
    check_quantized(quant, x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off,pad", [(0, 8), (1, 3), (8, 0), (3, 5)])
def test_quantize_rows_strided(quant, dtype, off, pad):
    base = torch.randn(9, 200 + off + pad, generator=rng(off), device="cuda").to(dtype)
    check_quantized(quant, base[:, off:off + 200])
    check_quantized(quant, base[::2, off:off + 199])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [5, 64, 4097])
def test_quantize_special_rows(quant, dtype, cols):
    x = torch.randn(8, cols, generator=rng(7), device="cuda").to(dtype)
    x[0] = 0
    x[1, cols // 2] = float("inf")
    x[2, cols - 1] = float("nan")
    x[3, 0] = float("-inf")
    x[3, 1] = float("nan")
    x[4] = torch.finfo(dtype).min
    x[5] *= 1e-38 if dtype != torch.float16 else 6e-8
    x[6] = -0.0
    x[7] = 0
    x[7, 2] = torch.finfo(dtype).tiny
    check_quantized(quant, x)


def linear_ref(q, s, w, ws, bias, gated):
    """(value, error of the 32-bit steps) in 64 bits, from int8 operands."""
    acc = q.double() @ w.double().t()
    y = acc * s.double()[:, None] * ws.double()
    dy = y.abs() * (3 * 2.0**-24)
    if bias is not None:
        y = y + bias.double()
        dy = dy + y.abs() * 2.0**-24
    if not gated:
        return y, dy
    n = y.shape[1] // 2
    g, u, dg, du = y[:, :n], y[:, n:], dy[:, :n], dy[:, n:]
    silu = g * torch.sigmoid(g)
    # |silu'| <= 1.1; exp (2 ulp), one addition, one division, one product.
    return silu * u, 1.1 * dg * u.abs() + silu.abs() * du + (silu * u).abs() * (8 * 2.0**-24)


def check_close(got, want, err, dtype):
    tol = err * 1.0 + want.abs() * U[dtype] * 1.01 + err * U[dtype] + TINY[dtype]
    d = (got.double() - want).abs()
    assert not torch.isnan(d).any()
    assert bool((d <= tol).all()), float((d / tol).max())


def operands(m, n, k, seed, ld_a=None, ld_w=None, off=0):
    g = rng(seed)

    def mat(r, c, ld):
        buf = torch.randint(-128, 128, (r * ld + off,), generator=g, device="cuda", dtype=torch.int16).to(torch.int8)
        return torch.as_strided(buf, (r, c), (ld, 1), off)

    a, w = mat(m, k, ld_a or k), mat(n, k, ld_w or k)
    s = torch.rand(m, generator=g, device="cuda") + 0.1
    ws = (torch.rand(n, generator=g, device="cuda") + 0.1) / 1000
    b = torch.randn(n, generator=g, device="cuda")
    return a, s, w, ws, b


SHAPES = [(1, 1, 1), (1, 16, 16), (1, 256, 4096), (2, 300, 1000), (3, 64, 15), (4, 513, 2064), (5, 100, 333),
          (8, 1000, 512), (9, 128, 128), (16, 384, 4096), (17, 129, 257), (31, 2048, 640), (33, 250, 96),
          (64, 512, 8192), (65, 100, 1040), (100, 1000, 1001), (128, 256, 256), (129, 257, 272), (200, 640, 4112),
          (256, 4096, 128), (257, 1024, 400), (511, 520, 1024), (1000, 1000, 1000), (1024, 2048, 144),
          (2048, 384, 2048), (1, 70000, 32), (3000, 8, 64), (40, 24, 131071), (2, 8, 131071)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm_scaled_shapes(quant, m, n, k, gated):
    a, s, w, ws, b = operands(m, 2 * n if gated else n, k, m * 7 + n + k)
    dtype = DTYPES[(m + n + k) % 3]
    if gated:  # keeps silu's argument in a range where f16 does not overflow
        s, b = s / k**0.5, b
    elif dtype == torch.float16:
        s = s / k**0.5
    bias = b if (m + k) % 2 else None
    got = quant.gemm_scaled(a, s, w, ws, bias=bias, gated=gated, out_dtype=dtype, quantize=False)
    assert got.shape == (m, n) and got.dtype == dtype
    check_close(got, *linear_ref(a, s, w, ws, bias, gated), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 4, 7, 40, 130, 700])
@pytest.mark.parametrize("ld_a,ld_w,off", [(1000, 1000, 0), (1008, 1024, 0), (1001, 1000, 1), (1008, 1008, 4),
                                           (1003, 1007, 3), (1016, 1008, 8)])
def test_gemm_scaled_strides(quant, m, ld_a, ld_w, off, dtype):
    a, s, w, ws, b = operands(m, 200, 1000, 11 * m + off, ld_a, ld_w, off)
    s = s / 32
    got = quant.gemm_scaled(a, s, w, ws, bias=b, out_dtype=dtype)
    check_close(got, *linear_ref(a, s, w, ws, b, False), dtype)


@pytest.mark.parametrize("m,n,k", [(1, 64, 131071), (6, 64, 131071), (48, 64, 131071), (300, 64, 131071)])
def test_gemm_scaled_extreme_sum(quant, m, n, k):
    """All operands -128: the sum is 128 * 128 * 131071, near the 32-bit limit."""
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[::2] = 127
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    got = quant.gemm_scaled(a, one_m, w, one_n, out_dtype=torch.float32)
    want = torch.full((m, n), 128.0 * 128 * k, dtype=torch.float64, device="cuda")
    want[:, ::2] = -128.0 * 127 * k
    check_close(got, want, want.abs() * 2.0**-24, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (2, 40, 77), (3, 300, 4096), (7, 256, 2048), (8, 64, 8192),
                                   (24, 512, 1000), (96, 300, 2048), (384, 1024, 520), (1500, 768, 256)])
def test_linear(quant, m, n, k, gated, dtype):
    g = rng(m + n + k)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    _, _, w, ws, b = operands(1, 2 * n if gated else n, k, n + k)
    ws = ws / k**0.5 * 4
    got = quant.linear(x, w, ws, bias=b, gated=gated)
    q, s = quantize_ref(x)
    want, err = linear_ref(torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), w, ws, b, gated)
    assert got.dtype == dtype
    check_close(got, want, err, dtype)
    # The one call equals its two steps bit for bit.
    two = quant.gemm_scaled(*quant.quantize_rows(x), w, ws, bias=b, gated=gated, out_dtype=dtype, quantize=False)
    assert torch.equal(got, two)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 512, 1024), (3, 40, 77), (48, 300, 4096), (200, 1001, 520),
                                   (1500, 768, 256)])
def test_quantized_result(quant, m, n, k, gated):
    """int8 rows out equal the quantisation, by its definition, of the 32-bit
    result; linear takes them as they are and answers in their type."""
    a, s, w, ws, b = operands(m, 2 * n if gated else n, k, m + n)
    s = s / k**0.5
    y = quant.gemm_scaled(a, s, w, ws, bias=b, gated=gated, out_dtype=torch.float32, quantize=False)
    rows = quant.gemm_scaled(a, s, w, ws, bias=b, gated=gated, out_dtype=torch.float16, quantize=True)
    q, scale = quantize_ref(y)
    assert rows.dtype == torch.float16 and rows.q.shape == (m, n)
    assert np.array_equal(rows.q.cpu().numpy(), q) and np.array_equal(rows.scale.cpu().numpy(), scale)
    assert torch.allclose(rows.dequantize().float(), y, rtol=0, atol=float(y.abs().max()) / 200)
    _, _, w2, ws2, _ = operands(1, 33, n, 3)
    ws2 = ws2 / 10
    out = quant.linear(rows, w2, ws2)
    assert out.dtype == torch.float16
    assert torch.equal(out, quant.gemm_scaled(rows.q, rows.scale, w2, ws2, out_dtype=torch.float16))
    assert torch.equal(out, quant.linear(y, w2, ws2, out_dtype=torch.float16))
    if gated:
        again = quant.gemm_scaled(a, s, w, ws, bias=b, gated=True)
        assert isinstance(again, quant.QuantizedRows) and again.dtype == torch.bfloat16 and torch.equal(again.q, rows.q)
    x = torch.randn(2, m, k, device="cuda")
    rows = quant.linear(x, w, ws, gated=gated, quantize=True)
    assert rows.q.shape == (2, m, n) and rows.scale.shape == (2, m)
    assert quant.linear(x[:, :0], w, ws, gated=gated, quantize=True).q.shape == (2, 0, n)


@pytest.mark.parametrize("m", [1, 3, 8, 20, 200])
@pytest.mark.parametrize("k", [64, 1000, 40000])
def test_linear_special_rows(quant, m, k):
    """A zero row gives the bias; a row with an infinity or NaN gives NaN and
    leaves the others alone."""
    x = torch.randn(m, k, generator=rng(k), device="cuda").to(torch.bfloat16)
    x[m - 1] = 0
    _, _, w, ws, b = operands(1, 48, k, k)
    got = quant.linear(x, w, ws, bias=b, out_dtype=torch.float32)
    assert torch.equal(got[m - 1], b)
    bad = x.clone()
    bad[0, k // 3] = float("nan") if m % 2 else float("inf")
    out = quant.linear(bad, w, ws, bias=b, out_dtype=torch.float32)
    assert torch.isnan(out[0]).all()
    assert torch.equal(out[1:], got[1:])


@pytest.mark.parametrize("m", [1, 4, 60, 400])
@pytest.mark.parametrize("off,pad", [(0, 8), (1, 0), (3, 2)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_strided_activations(quant, m, off, pad, dtype):
    k = 520
    base = torch.randn(m, k + off + pad, generator=rng(m), device="cuda").to(dtype)
    x = base[:, off:off + k]
    _, _, w, ws, b = operands(1, 96, k, 5)
    assert torch.equal(quant.linear(x, w, ws, bias=b), quant.linear(x.contiguous(), w, ws, bias=b))


def test_leading_dimensions_and_empty_batches(quant):
    _, _, w, ws, b = operands(1, 64, 128, 3)
    x = torch.randn(2, 3, 128, generator=rng(1), device="cuda")
    assert torch.equal(quant.linear(x, w, ws), quant.linear(x.view(6, 128), w, ws).view(2, 3, 64))
    assert torch.equal(quant.linear(x[0, 0], w, ws), quant.linear(x[0, :1], w, ws)[0])
    q, s = quant.quantize_rows(x)
    assert q.shape == (2, 3, 128) and s.shape == (2, 3)
    assert torch.equal(quant.gemm_scaled(q, s, w, ws, out_dtype=torch.float32), quant.linear(x, w, ws))
    assert quant.linear(x[:0], w, ws).shape == (0, 3, 64)
    assert quant.gemm_scaled(q[:0], s[:0], w, ws).shape == (0, 3, 64)
    assert quant.quantize_rows(x.view(6, 128)[:0])[0].shape == (0, 128)


def test_output_leading_dimension_and_offsets_past_32_bits(quant):
    """Rows of the output (and of the activations) 3e9 bytes apart, through the
    C entry; what lies between rows is untouched."""
    from rns8_b200 import abi

    m, n, k, ld = 3, 40, 64, 1_500_000_000
    a, s, w, ws, b = operands(m, n, k, 21)
    far_a = torch.empty(2 * ld + k, dtype=torch.int8, device="cuda")
    view_a = torch.as_strided(far_a, (m, k), (ld, 1))
    view_a.copy_(a)
    out = torch.zeros(2 * ld + n + 8, dtype=torch.bfloat16, device="cuda")
    d = abi.LinearDesc()
    d.a_type, d.m, d.n, d.k, d.ld_a, d.ld_w, d.ld_out = 3, m, n, k, ld, k, ld
    d.a, d.a_scale, d.w, d.w_scale, d.bias, d.out = (t.data_ptr() for t in (view_a, s, w, ws, b, out))
    d.status, d.stream = quant.device_status(0).data_ptr(), torch.cuda.current_stream().cuda_stream
    need = abi.lib().rns8_cuda_linear_scratch_bytes(C.byref(d))
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    d.scratch, d.scratch_bytes = scratch.data_ptr(), need
    assert abi.lib().rns8_cuda_linear_device(C.byref(d)) == 0
    got = torch.as_strided(out, (m, n), (ld, 1))
    check_close(got, *linear_ref(a, s, w, ws, b, False), torch.bfloat16)
    assert int(torch.count_nonzero(out[n:n + 4096])) == 0 and int(torch.count_nonzero(out[ld - 4096:ld])) == 0
    assert int(torch.count_nonzero(out[2 * ld + n:])) == 0


@pytest.mark.parametrize("m", [5, 150])
def test_scratch_too_small_is_refused(quant, m):
    from rns8_b200 import abi

    x = torch.ones(m, 35, dtype=torch.bfloat16, device="cuda")
    _, _, w, ws, _ = operands(1, 33, 35, 2)
    out = torch.zeros(m, 33, dtype=torch.bfloat16, device="cuda")
    d = abi.LinearDesc()
    d.m, d.n, d.k, d.ld_a, d.ld_w, d.ld_out = m, 33, 35, 35, 35, 33
    d.a, d.w, d.w_scale, d.out = (t.data_ptr() for t in (x, w, ws, out))
    d.status, d.stream = quant.device_status(0).data_ptr(), torch.cuda.current_stream().cuda_stream
    need = abi.lib().rns8_cuda_linear_scratch_bytes(C.byref(d))
    assert need > 0
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    d.scratch, d.scratch_bytes = scratch.data_ptr(), need - 1
    assert abi.lib().rns8_cuda_linear_device(C.byref(d)) == 7
    torch.cuda.synchronize()
    assert int(torch.count_nonzero(out)) == 0


@pytest.mark.parametrize("m", [1, 50, 600])
def test_other_stream_graph_and_repeat(quant, m):
    g = rng(m)
    x = torch.randn(m, 1024, generator=g, device="cuda").to(torch.bfloat16)
    _, _, w, ws, b = operands(1, 512, 1024, 9)
    want = quant.linear(x, w, ws, bias=b)
    for _ in range(5):
        assert torch.equal(quant.linear(x, w, ws, bias=b), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = quant.linear(x, w, ws, bias=b)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = quant.linear(x, w, ws, bias=b)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, quant.linear(x, w, ws, bias=b))
    quant.check_status(0)


def test_python_refusals(quant):
    x = torch.zeros(4, 32, device="cuda")
    w = torch.zeros(8, 32, dtype=torch.int8, device="cuda")
    ws = torch.ones(8, device="cuda")
    with pytest.raises(ValueError):
        quant.linear(x[:, :31], w, ws)
    with pytest.raises(TypeError):
        quant.linear(x, w.float(), ws)
    with pytest.raises(TypeError):
        quant.linear(x, w, ws[:7])
    with pytest.raises(TypeError):
        quant.linear(x, w, ws.double())
    with pytest.raises(TypeError):
        quant.linear(x, w, ws, bias=ws.half())
    with pytest.raises(TypeError):
        quant.linear(x.double(), w, ws)
    with pytest.raises(TypeError):
        quant.linear(x, w, ws, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        quant.linear(x, w[:7], ws[:7], gated=True)
    with pytest.raises(ValueError):
        quant.linear(x, w.cpu(), ws)
    with pytest.raises(ValueError):
        quant.linear(x.t(), w[:, :4], ws)
    with pytest.raises(TypeError):
        quant.gemm_scaled(w, ws[:7], w, ws)
    from rns8_b200 import Error

    big = torch.zeros(1, 131072, dtype=torch.int8, device="cuda")
    with pytest.raises(Error) as e:
        quant.gemm_scaled(big, ws[:1], big, ws[:1])
    assert e.value.status == 6
