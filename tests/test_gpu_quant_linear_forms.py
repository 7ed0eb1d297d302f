"""Every kernel form of the scaled int8 product: tokens or channels on the
tensor cores' lanes, each number of tokens to a tile, each number of blocks that
share k, gated and not, for each output type. The shapes leave a remainder in
every direction. Formulas and error model are those of test_gpu_quant_linear."""

import ctypes as C

import pytest

from test_gpu_quant_linear import DTYPES, check_close, linear_ref, operands

torch = pytest.importorskip("torch")

# (gated, tokens to a tile or 0 for tokens on lanes, blocks to a cluster) -> m, n, k
# on 148 multiprocessors. Tokens on lanes: more than two tiles a multiprocessor
# and several rings of k a tile.
FORMS = {
    (False, 0, 1): (2500, 8200, 1104), (False, 16, 1): (1, 201, 64), (False, 16, 2): (2, 204, 400),
    (False, 16, 4): (2, 202, 912), (False, 16, 8): (5, 202, 1936), (False, 32, 1): (1685, 261, 64),
    (False, 32, 2): (1157, 232, 1088), (False, 32, 4): (613, 208, 944), (False, 32, 8): (165, 234, 1936),
    (False, 64, 1): (3400, 281, 64), (False, 64, 2): (1068, 425, 1712), (False, 64, 4): (735, 257, 1008),
    (False, 64, 8): (197, 259, 1936), (False, 128, 1): (6536, 273, 64), (False, 128, 2): (2845, 268, 3392),
    (False, 128, 4): (2221, 207, 2000), (False, 128, 8): (431, 261, 3920), (False, 256, 8): (771, 290, 9120),
    (True, 0, 1): (2500, 4100, 1104), (True, 16, 1): (1, 200, 64), (True, 16, 2): (3, 203, 400),
    (True, 16, 4): (2, 205, 912), (True, 16, 8): (8, 200, 1952), (True, 32, 1): (1277, 202, 272),
    (True, 32, 2): (571, 217, 400), (True, 32, 4): (286, 213, 960), (True, 32, 8): (77, 217, 2016),
    (True, 64, 1): (4359, 202, 2656), (True, 64, 2): (839, 257, 704), (True, 64, 4): (541, 211, 1200),
    (True, 64, 8): (149, 203, 1968), (True, 128, 1): (6770, 263, 1680), (True, 128, 2): (2213, 202, 1200),
    (True, 128, 4): (890, 269, 1984), (True, 128, 8): (304, 201, 3952), (True, 256, 8): (607, 204, 8784),
}
# The persistent form again: few columns of many token tiles (past one group of
# 32), and few token tiles of many columns.
MORE = [(False, (8515, 1070, 608)), (False, (390, 40000, 616)), (True, (268, 15265, 656)), (True, (8515, 523, 1160))]


def form(rns8, m, n, k, gated, sms=148):
    d = rns8.abi.LinearDesc()
    d.a_type, d.flags, d.m, d.n, d.k, d.ld_a, d.ld_w, d.ld_out = 3, int(gated), m, n, k, k, k, n
    d.a = d.a_scale = d.w = d.w_scale = d.out = 4096  # never read
    tile, splits = C.c_uint32(), C.c_uint32()
    assert rns8.lib().rns8_cuda_linear_form(C.byref(d), sms, C.byref(tile), C.byref(splits)) == 0
    return tile.value, splits.value


def test_the_shapes_cover_every_form(rns8):
    for key, shape in FORMS.items():
        assert form(rns8, *shape, key[0]) == key[1:], (key, shape)
    for gated, shape in MORE:
        assert form(rns8, *shape, gated) == (0, 1), shape
    kernels = {key[:2] for key in FORMS}
    assert kernels == {(g, t) for g in (False, True) for t in (0, 16, 32, 64, 128, 256)}
    # And nothing else is ever chosen.
    for gated in (False, True):
        for m in (1, 5, 16, 24, 48, 100, 150, 256, 300, 520, 900, 1500, 2500, 4096, 8192, 30000):
            for n in (8, 100, 512, 768, 1024, 3000, 4096, 11008, 16384, 70000):
                for k in (16, 144, 512, 1024, 2064, 4096, 8192, 16384, 70000, 131071):
                    assert (gated, *form(rns8, m, n, k, gated)) in FORMS, (m, n, k, gated)


def test_form_refusals(rns8):
    d = rns8.abi.LinearDesc()
    d.a_type, d.m, d.n, d.k, d.ld_a, d.ld_w, d.ld_out = 3, 4, 8, 16, 16, 16, 8
    d.a = d.a_scale = d.w = d.w_scale = d.out = 4096
    tile, splits = C.c_uint32(), C.c_uint32()
    ask = rns8.lib().rns8_cuda_linear_form
    assert ask(C.byref(d), 148, C.byref(tile), C.byref(splits)) == 0
    assert ask(C.byref(d), 0, C.byref(tile), C.byref(splits)) == 1
    assert ask(C.byref(d), 148, None, C.byref(splits)) == 1 and ask(C.byref(d), 148, C.byref(tile), None) == 1
    assert ask(None, 148, C.byref(tile), C.byref(splits)) == 1
    d.m = 0
    assert ask(C.byref(d), 148, C.byref(tile), C.byref(splits)) == 1


def check(quant, m, n, k, gated, dtype, bias):
    a, s, w, ws, b = operands(m, 2 * n if gated else n, k, m + n + k)
    s = s / k**0.5  # in f16's range
    b = b if bias else None
    got = quant.gemm_scaled(a, s, w, ws, bias=b, gated=gated, out_dtype=dtype, quantize=False)
    assert got.shape == (m, n) and got.dtype == dtype
    check_close(got, *linear_ref(a, s, w, ws, b, gated), dtype)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("key", FORMS)
def test_every_form(rns8, key, dtype):
    from rns8_b200 import quant

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    m, n, k = FORMS[key]
    if sms == 148:
        assert form(rns8, m, n, k, key[0]) == key[1:]
    first = check(quant, m, n, k, key[0], dtype, True)
    assert torch.equal(check(quant, m, n, k, key[0], dtype, True), first)
    check(quant, m, n, k, key[0], dtype, False)
    check(quant, m, n - n % 8, k, key[0], dtype, True)  # rows of whole words out
    quant.check_status(0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated,shape", MORE)
def test_persistent_form(gated, shape, dtype):
    from rns8_b200 import quant

    check(quant, *shape, gated, dtype, True)
    quant.check_status(0)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_persistent_form_behind_its_quantiser_and_into_int8(gated):
    """Float tokens in and int8 rows out equal the steps one by one."""
    from rns8_b200 import quant

    m, n, k = 2500, 4100 if gated else 8200, 1104
    _, _, w, ws, b = operands(1, 2 * n if gated else n, k, 5)
    ws = ws / k**0.5
    x = torch.randn(m, k, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(torch.bfloat16)
    y = quant.linear(x, w, ws, bias=b, gated=gated, out_dtype=torch.float32)
    q, s = quant.quantize_rows(x)
    check_close(y, *linear_ref(q, s, w, ws, b, gated), torch.float32)
    rows = quant.linear(x, w, ws, bias=b, gated=gated, quantize=True)
    wq, wscale = quant.quantize_rows(y)
    assert torch.equal(rows.q, wq) and torch.equal(rows.scale, wscale)
