"""The 8-bit dense layer: codes and scales bit for bit those of the definition, products of integers exact, the rest to the bound of dense_util.fp8_reference."""
import pytest
import torch

from dense_util import assert_within, fp8_reference, fp8_rows, fp8_weight, ints, normals
from mortar_amd import ops

pytestmark = pytest.mark.gpu


def _bits(q):
    return q.view(torch.uint8)


@pytest.mark.parametrize("M,K", [(1, 16), (3, 128), (5, 144), (17, 400), (64, 2048), (130, 1360), (1003, 272)])
def test_codes_of_activations(dev, M, K):
    x = normals((M, K), M + K, torch.bfloat16, dev) * torch.exp2(torch.randint(-30, 30, (M, 1), device=dev).float()).bfloat16()
    x[:, ::17] *= 20
    x[0, :128] = 0                                        # a group of zeros has the scale 1
    x[-1, -16:] = torch.tensor([3e-39, 1e-38, -2e-39, 0] * 4, dtype=torch.bfloat16)
    if M > 2:
        x[1] = 1e-38                                      # the smallest normal values and below
        x[2, ::2] = -3.3e38                               # the largest
    q, s = ops.quantize_fp8(x)
    rq, rs = fp8_rows(x.cpu())
    assert torch.equal(s.cpu(), rs) and torch.equal(_bits(q).cpu(), _bits(rq))
    assert s.shape == (M, -(-K // 128)) and s.stride(0) == 1 or M == 1


def test_quotients_near_ties(dev):
    """Every bf16 pattern of two octaves against many scales: the fp32 quotient's rounding decides, not a reciprocal's."""
    m = torch.arange(256, dtype=torch.int32)
    vals = ((m + 0x3F80).to(torch.int16)).view(torch.bfloat16)                # 1 .. 4
    x = torch.zeros((997, 272), dtype=torch.bfloat16)
    x[:, :127] = vals[:254:2]
    x[:, 128:255] = vals[1:255:2]
    top = ((torch.arange(997, dtype=torch.int32) * 3 + 0x4090).to(torch.int16)).view(torch.bfloat16)
    x[:, 127], x[:, 255] = top, -top
    q, s = ops.quantize_fp8(x.to(dev))
    rq, rs = fp8_rows(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(_bits(q).cpu(), _bits(rq))


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("N,K", [(1, 16), (8, 128), (128, 128), (130, 400), (264, 272), (1000, 2048)])
def test_codes_of_weights(dev, N, K, t):
    w = normals((N, K), N, torch.float32, dev, K ** -0.5).to(t)
    w[: N // 2, : K // 2] *= 100
    if N > 128:
        w[128:, 128:256] = 0
    q, s = ops.quantize_fp8_weight(w)
    rq, rs = fp8_weight(w.cpu())
    assert torch.equal(s.cpu(), rs) and torch.equal(_bits(q).cpu(), _bits(rq))
    wide = torch.zeros((N, K + 24), dtype=t, device=dev)
    for view in (wide[:, 8:8 + K], wide[:, 5:5 + K]):
        view.copy_(w)
        assert torch.equal(_bits(ops.quantize_fp8_weight(view)[0]), _bits(q))


SIZES = [(1, 8, 16), (2, 24, 128), (7, 136, 272), (16, 264, 1360), (16, 128, 2048), (17, 136, 400), (33, 256, 144), (64, 520, 1040), (65, 8, 16), (130, 264, 400), (300, 136, 2736), (520, 1032, 272),
         (2100, 2056, 400), (70, 64, 8192), (20, 2056, 4112)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_products_of_integers_are_exact(dev, M, N, K):
    """Codes that are small integers and scales that are powers of two: every sum is exact, the result its rounding."""
    xq, wq = ints((M, K), 3, M, torch.float32, dev).to(torch.float8_e4m3fn), ints((N, K), 3, N + 1, torch.float32, dev).to(torch.float8_e4m3fn)
    kb, nb = -(-K // 128), -(-N // 128)
    xs, ws = torch.exp2(ints((M, kb), 2, 5, torch.float32, dev)), torch.exp2(ints((nb, kb), 2, 6, torch.float32, dev))
    want = fp8_reference(xq, xs, wq, ws)[0].bfloat16()
    assert torch.equal(ops.linear_fp8(xq, wq, ws, xs), want)
    assert torch.equal(ops.linear_fp8(xq, wq, ws, xs.t().contiguous().t()), want)
    wide = torch.zeros((M, K + 32), dtype=torch.uint8, device=dev)
    wide[:, 16:16 + K] = xq.view(torch.uint8)
    ww = torch.zeros((N, K + 16), dtype=torch.uint8, device=dev)
    ww[:, :K] = wq.view(torch.uint8)
    assert torch.equal(ops.linear_fp8(wide[:, 16:16 + K].view(torch.float8_e4m3fn), ww[:, :K].view(torch.float8_e4m3fn), ws, xs), want)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(dev, M, N, K):
    x = normals((M, K), M, torch.bfloat16, dev)
    x[:, ::50] *= 16
    wq, ws = ops.quantize_fp8_weight(normals((N, K), N, torch.float32, dev, K ** -0.5))
    y = ops.linear_fp8(x, wq, ws)
    xq, xs = fp8_rows(x.cpu())
    xq, xs = xq.to(dev), xs.to(dev)
    ref, bound = fp8_reference(xq, xs, wq, ws)
    assert y.dtype == torch.bfloat16
    assert_within(y, ref, bound, "y")
    assert torch.equal(ops.linear_fp8(*ops.quantize_fp8(x)[:1], wq, ws, ops.quantize_fp8(x)[1]), y)
    assert float((y.double() - ref).norm() / ref.norm()) <= 2.0 ** -8 / 3 ** 0.5       # no more than one rounding to bf16 is off by on average


def test_a_few_rows_do_not_depend_on_who_quantises(dev):
    wq, ws = ops.quantize_fp8_weight(normals((264, 2048), 1, torch.float32, dev, 0.02))
    x = normals((16, 2048), 2, torch.bfloat16, dev)
    q, s = ops.quantize_fp8(x)
    for M in range(1, 17):
        assert torch.equal(ops.linear_fp8(x[:M], wq, ws), ops.linear_fp8(q[:M], wq, ws, s[:M]))


def test_shapes_strides_and_no_rows(dev):
    wq, ws = ops.quantize_fp8_weight(normals((72, 160), 1, torch.float32, dev, 0.1))
    x = normals((12, 160), 2, torch.bfloat16, dev)
    y = ops.linear_fp8(x, wq, ws)
    assert torch.equal(ops.linear_fp8(x.view(3, 4, 160), wq, ws), y.view(3, 4, 72)) and torch.equal(ops.linear_fp8(x[5], wq, ws), y[5])
    wide = torch.full((12, 400), float("nan"), dtype=torch.bfloat16, device=dev)
    for view in (wide[:, 8:168], wide[:, 3:163], wide[:, 40:360:2]):
        view.copy_(x)
        assert torch.equal(ops.linear_fp8(view, wq, ws), y)
    q, s = ops.quantize_fp8(x.view(3, 4, 160))
    assert q.shape == (3, 4, 160) and s.shape == (3, 4, 2) and torch.equal(ops.linear_fp8(q, wq, ws, s), y.view(3, 4, 72))
    assert torch.equal(ops.linear_fp8(x, wq, ws.t().contiguous().t()), y)
    assert ops.linear_fp8(x[:0], wq, ws).shape == (0, 72)
    q, s = ops.quantize_fp8(x[:0])
    assert q.shape == (0, 160) and s.shape == (0, 2)


def test_rows_that_are_not_finite_stay_among_themselves(dev):
    wq, ws = ops.quantize_fp8_weight(normals((72, 400), 1, torch.float32, dev, 0.1))
    for M in (9, 100):
        x = normals((M, 400), 2, torch.bfloat16, dev)
        good = ops.linear_fp8(x, wq, ws)
        x[3, 5], x[6, 399], x[M - 1, 130] = float("nan"), float("inf"), float("-inf")
        y = ops.linear_fp8(x, wq, ws)
        bad = [3, 6, M - 1]
        keep = [i for i in range(M) if i not in bad]
        assert torch.equal(y[keep], good[keep]) and bool(y[bad].isnan().all())


def test_replayed_from_a_graph(dev):
    wq, ws = ops.quantize_fp8_weight(normals((264, 272), 1, torch.float32, dev, 0.1))
    for M in (4, 40, 200):
        x = normals((M, 272), 3, torch.bfloat16, dev)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.linear_fp8(x, wq, ws)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear_fp8(x, wq, ws)
        for i in range(3):
            x.copy_(normals((M, 272), 10 + i, torch.bfloat16, dev))
            g.replay()
            want = ops.linear_fp8(x, wq, ws)
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_refusals(dev):
    x = normals((4, 160), 2, torch.bfloat16, dev)
    wq, ws = ops.quantize_fp8_weight(normals((72, 160), 1, torch.float32, dev, 0.1))
    q, s = ops.quantize_fp8(x)
    with pytest.raises(TypeError):
        ops.linear_fp8(x.float(), wq, ws)
    with pytest.raises(TypeError):
        ops.linear_fp8(q, wq, ws)
    with pytest.raises(TypeError):
        ops.linear_fp8(x, wq, ws, s)
    with pytest.raises(TypeError):
        ops.linear_fp8(x, wq.float(), ws)
    with pytest.raises(ValueError):
        ops.linear_fp8(x[:, :144], wq, ws)
    with pytest.raises(ValueError):
        ops.linear_fp8(x, wq, ws[:, :1])
    with pytest.raises(ValueError):
        ops.linear_fp8(q, wq, ws, s[:, :1])
    with pytest.raises(ValueError):
        ops.linear_fp8(x, wq[:68], ws)
    with pytest.raises(ValueError):
        ops.quantize_fp8(x[:, :152])
    with pytest.raises(TypeError):
        ops.quantize_fp8(x.half())
    with pytest.raises(RuntimeError):
        ops.linear_fp8(x, wq.cpu(), ws)
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.linear_fp8(x.clone().requires_grad_(True), wq, ws)
    with torch.no_grad():
        ops.linear_fp8(x.clone().requires_grad_(True), wq, ws)
