"""Every form of the dense products: each tile in each operand layout and epilogue, with and without ranges of K, over enough steps that the ring
of copies runs round, in sizes that end inside tiles; and the kernels of few rows up to where tiles take over.  What the host chooses is asserted, so
that a changed estimate cannot leave a form out.  Integers, whose sums are exact."""
import pytest
import torch

from dense_util import assert_within, fp8_reference, ints, normals, rounding
from mortar_amd import _lib, ops
from test_gpu_dense_mlp import TYPES, _bytes24, _padded, _product, _stream, _values24
from util import dense_form

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
LINEAR, TRANSPOSED, GATE_UP, GATE_UP_KEPT, SWIGLU_BWD, E4M3 = range(6)


def _swiglu(exact, t):
    """h = g sigmoid(g) u of exact gate and up values, and its bound: eight fp32 steps and one rounding.  For g < -126 ln 2 = -87.3 the sigmoid lies
    below 2^-126, the smallest normal fp32 value, where the reciprocal gives 0 (and 1 + exp(-g) is infinite from -88.7 on, for torch too): off
    by no more than itself, so h by no more than |h|, which is then below 2^-126 |g u|."""
    g, u = exact.chunk(2, 1)
    s = torch.sigmoid(g)
    ref = g * s * u
    return ref, rounding(t, ref) + torch.where(s < 2.0 ** -126, ref.abs(), 8 * 2.0 ** -23 * ref.abs())


#          M, N, K (K - 3 where K is a number of rows), tile of N x M, ranges
PRODUCTS = [(77, 72, 584, (64, 64), 1), (7, 1080, 7248, (64, 64), 12), (8413, 208, 592, (128, 128), 1), (8723, 72, 1760, (128, 128), 3), (389, 8728, 672, (256, 128), 1),
            (67, 8576, 3488, (256, 128), 6), (8429, 904, 592, (256, 192), 1), (141, 7080, 4976, (256, 192), 8), (4617, 2592, 592, (256, 256), 1), (401, 5400, 4144, (256, 256), 5)]
PRODUCTS_T = [(80, 72, 584, (64, 64), 1), (8, 4128, 1752, (64, 64), 3), (6632, 264, 624, (128, 128), 1), (72, 4272, 3680, (128, 128), 6), (648, 5920, 576, (256, 128), 1),
              (2736, 136, 6224, (256, 128), 10), (928, 8712, 592, (256, 192), 1), (136, 4200, 7712, (256, 192), 12), (1552, 7632, 592, (256, 256), 1), (8464, 264, 5200, (256, 256), 3)]


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("form,case", [("y", c) for c in PRODUCTS] + [(f, c) for f in ("dx", "dw") for c in PRODUCTS_T], ids=str)
def test_plain_products(dev, form, case, t):
    M, N, K, tile, ranges = case
    if form == "dw":
        K -= 3
    if form == "y" and M <= 8:
        M = 9                                            # (fewer are those of the other kernel)
    elif form == "dx" and M > 8:
        M -= 3
    assert dense_form(LINEAR if form == "y" else TRANSPOSED, M, N, K) == (tile, ranges)
    for extra in (0, 8):
        c, exact, intact = _product(form, M, N, K, t, dev, 7, extra)
        assert torch.equal(c, exact.to(t)) and intact


GATE_UPS = [(77, 72, 584, (64, 64)), (66, 8992, 584, (128, 128)), (152, 8488, 624, (256, 128)), (520, 7240, 592, (256, 192)), (7184, 800, 584, (256, 256)),
            (77, 72, 584, (64, 64)), (68, 8496, 672, (128, 128)), (130, 8248, 880, (256, 128)), (535, 7424, 584, (256, 192)), (603, 8400, 584, (256, 256))]


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("kept,case", list(zip([False] * 5 + [True] * 5, GATE_UPS)), ids=str)
def test_gate_up(dev, kept, case, t):
    """Kept gate and up values exact, h to the bound of _swiglu."""
    M, f, d, tile = case
    assert dense_form(GATE_UP_KEPT if kept else GATE_UP, M, f, d) == (tile, 1)
    x, w = ints((M, d), 1, M, t, dev), ints((2 * f, d), 1, f, t, dev)
    hw, h = _padded(M, f, 8, t, dev)
    gu = torch.full((6 * M * f + 16,), 0xAB, dtype=torch.uint8, device=dev)
    _lib.check(_lib.lib().mortar_dense_gateup_swiglu(x.data_ptr(), M, d, d, w.data_ptr(), d, f, TYPES[t], h.data_ptr(), h.stride(0), gu.data_ptr() if kept else None, _stream()),
               "gateup")
    exact = x.double() @ w.double().t()
    assert_within(h, *_swiglu(exact, t), "h")
    assert bool(hw[M:].isnan().all() and hw[:M, f:].isnan().all())
    if kept:
        assert torch.equal(_values24(gu, M, 2 * f), exact) and bool((gu[6 * M * f:] == 0xAB).all())


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("case", [(77, 72, 584, (64, 64)), (4430, 688, 584, (128, 128)), (7608, 520, 768, (256, 128)), (23116, 264, 584, (256, 192)), (1029, 11136, 4416, (256, 256))], ids=str)
def test_gradient_in_the_epilogue(dev, case, t):
    """dh exact, the derivative and h ten fp32 steps and one rounding; every row's gate and up are its own."""
    M, f, d, tile = case
    assert dense_form(SWIGLU_BWD, M, f, d) == (tile, 1)
    dy, w = ints((M, d), 1, M, t, dev), ints((d, f), 1, f, t, dev)
    gu = normals((M, 2 * f), 3, torch.float32, dev, 2.0)
    gu = (gu.view(torch.int32) & ~0xff).view(torch.float32)
    kept = _bytes24(gu)
    dh = dy.double() @ w.double()
    g, u = gu.double().chunk(2, 1)
    s = torch.sigmoid(g)
    ref = torch.cat([dh * u * s * (1 + g * (1 - s)), dh * g * s], 1)
    size = torch.cat([(dh * u).abs() * (s + (g * s * (1 - s)).abs()), (dh * g * s).abs()], 1)
    hr = g * s * u
    step = 10 * 2.0 ** -23
    for want_h in (True, False):
        ow, dgu = _padded(M, 2 * f, 8, t, dev)
        hw, h = _padded(M, f, 8, t, dev)
        _lib.check(_lib.lib().mortar_dense_swiglu_bwd(dy.data_ptr(), M, d, d, w.data_ptr(), f, f, TYPES[t], kept.data_ptr(), dgu.data_ptr(), dgu.stride(0),
                                                      h.data_ptr() if want_h else None, h.stride(0), _stream()), "swiglu_bwd")
        assert_within(dgu, ref, rounding(t, ref) + step * size, "dgu")
        assert bool(ow[M:].isnan().all() and ow[:M, 2 * f:].isnan().all())
        if want_h:
            assert_within(h, hr, rounding(t, hr) + step * hr.abs(), "h")
            assert bool(hw[M:].isnan().all() and hw[:M, f:].isnan().all())
        else:
            assert bool(hw.isnan().all())


# (from 2^24 results on they are stored past the caches)
@pytest.mark.parametrize("case", [(77, 72, 1360, (64, 64), 1), (17, 5944, 2592, (64, 64), 2), (8266, 208, 1184, (128, 128), 1), (130, 2224, 7344, (128, 128), 6),
                                  (6563, 592, 5136, (256, 128), 1), (1678, 4880, 3120, (256, 192), 1), (6567, 528, 6672, (256, 192), 2), (4093, 11256, 2064, (128, 128), 1),
                                  (4091, 4104, 1296, (128, 128), 1), (5003, 4104, 4112, (256, 192), 1)], ids=str)
def test_8_bit_products(dev, case):
    M, N, K, tile, ranges = case
    assert dense_form(E4M3, M, N, K) == (tile, ranges)
    xq, wq = ints((M, K), 3, M, torch.float32, dev).to(torch.float8_e4m3fn), ints((N, K), 3, N + 1, torch.float32, dev).to(torch.float8_e4m3fn)
    kb, nb = -(-K // 128), -(-N // 128)
    xs, ws = torch.exp2(ints((M, kb), 2, 5, torch.float32, dev)), torch.exp2(ints((nb, kb), 2, 6, torch.float32, dev))
    assert torch.equal(ops.linear_fp8(xq, wq, ws, xs), fp8_reference(xq, xs, wq, ws)[0].to(BF16))


# ---- few rows


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("N,K", [(8, 8), (24, 72), (264, 1000), (1048, 2736), (88, 5632)])
def test_few_rows(dev, N, K, t):
    for M in range(1, 10):
        assert (dense_form(LINEAR, M, N, K)[0] == (0, 0)) == (M <= 8)
        for extra in (0, 8):
            c, exact, intact = _product("y", M, N, K, t, dev, M + N, extra)
            assert torch.equal(c, exact.to(t)) and intact, (M, extra)


@pytest.mark.parametrize("M,K", [(8, 6016), (8, 6024), (8, 6144), (8, 6152), (5, 9720), (5, 9856), (1, 48000), (1, 49152)])
def test_few_rows_that_are_long(dev, M, K):
    """On both sides of what the kernel's LDS holds: M (256 ceil(K / 128) + 16) bytes in 96 KB."""
    few = M * (-(-K // 128) * 256 + 16) <= 96 * 1024
    assert (dense_form(LINEAR, M, 72, K)[0] == (0, 0)) == few
    c, exact, intact = _product("y", M, 72, K, BF16, dev, M)
    assert torch.equal(c, exact.to(BF16)) and intact


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("d,f", [(8, 8), (64, 40), (1000, 72), (2048, 264)])
def test_few_rows_of_gate_up(dev, d, f, t):
    for M in range(1, 10):
        x, w = ints((M, d), 1, M, t, dev), ints((2 * f, d), 1, f, t, dev)
        for kept in (True, False):
            assert (dense_form(GATE_UP_KEPT if kept else GATE_UP, M, f, d)[0] == (0, 0)) == (M <= 8)
            hw, h = _padded(M, f, 8, t, dev)
            gu = torch.full((6 * M * f + 16,), 0xAB, dtype=torch.uint8, device=dev)
            _lib.check(_lib.lib().mortar_dense_gateup_swiglu(x.data_ptr(), M, d, d, w.data_ptr(), d, f, TYPES[t], h.data_ptr(), h.stride(0), gu.data_ptr() if kept else None,
                                                             _stream()), "gateup")
            exact = x.double() @ w.double().t()
            assert_within(h, *_swiglu(exact, t), "h")
            assert bool(hw[M:].isnan().all() and hw[:M, f:].isnan().all())
            assert torch.equal(_values24(gu, M, 2 * f), exact) and bool((gu[6 * M * f:] == 0xAB).all()) if kept else bool((gu == 0xAB).all())
