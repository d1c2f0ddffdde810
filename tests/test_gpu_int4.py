"""The 4-bit dense layer: codes by their definition, products of integers exact, the rest within the bound of operators_util.int4_bound and as near as rounding."""
import pytest
import torch

from dense_util import assert_within, ints, normals
from mortar_amd import ops
from operators_util import INT4_SIZES, int4_bound, int4_weight, pack_codes, quantize_reference, unpack_codes

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (3, 31, 64), (16, 128, 128), (17, 130, 32), (130, 400, 64), (264, 1999, 128)])
def test_codes_of_weights(dev, N, K, group, t, zeros):
    w = normals((N, K), N + K, torch.float32, dev, K ** -0.5).to(t)
    if N > 2:
        w[1] = 0                                         # scale 1, codes of the zero point
        w[2] = w[2].abs() + 1                            # of one sign: 0 is in the range all the same
    c, s, z = ops.quantize_int4_weight(w, group, zeros)
    rq, rs, rz = quantize_reference(w.cpu(), group, zeros)
    assert torch.equal(s.cpu(), rs) and (z is None) == (rz is None) and (z is None or torch.equal(z.cpu(), rz))
    assert torch.equal(c.cpu(), pack_codes(rq)) and s.stride(0) == 1
    wide = torch.zeros((N, K + 24), dtype=t, device=dev)
    wide[:, 5:5 + K] = w
    assert torch.equal(ops.quantize_int4_weight(wide[:, 5:5 + K], group, zeros)[0], c)
    assert torch.equal(ops.quantize_int4_weight(w.t().contiguous().t(), group, zeros)[0], c)


def test_weights_that_are_not_finite(dev):
    """A group with an infinity or NaN makes its row NaN, and no other."""
    w = normals((9, 256), 0, torch.bfloat16, dev)
    w[3, 7], w[5, 200] = float("nan"), float("-inf")
    c, s, z = ops.quantize_int4_weight(w, 128)
    y = ops.linear_int4(normals((2, 256), 1, torch.bfloat16, dev), c, s)
    assert torch.equal(torch.isnan(y).any(0).cpu(), torch.tensor([i in (3, 5) for i in range(9)]))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,N,K", INT4_SIZES)
def test_products_of_integers_are_exact(dev, M, N, K, t, group, zeros):
    """Small integers in x and powers of two as scales: every sum is exact in fp32 (K 31 3 4 below 2^24), the result its rounding."""
    x = ints((M, K), 2, M + K, t, dev)
    q = torch.randint(0, 16, (N, K), generator=torch.Generator().manual_seed(N)).to(dev)
    groups = -(-K // group)
    s = torch.exp2(ints((N, groups), 1, 5, torch.float32, dev)).to(t)
    z = torch.randint(0, 16, (N, groups), generator=torch.Generator().manual_seed(7), dtype=torch.uint8).to(dev) if zeros else None
    c = pack_codes(q)
    want = (x.double() @ int4_weight(c, s, z, group, K).t()).to(t)
    assert torch.equal(ops.linear_int4(x, c, s, z, group), want)
    zc = z if z is None else z.t().contiguous().t()
    assert torch.equal(ops.linear_int4(x, c, s.t().contiguous().t().float(), zc, group), want)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,N,K", [(1, 264, 2048), (16, 2048, 5632), (20, 520, 1999), (77, 1031, 1040), (1000, 1040, 2056), (2100, 2056, 392), (4200, 131, 4104)])
def test_products(dev, M, N, K, t, group, zeros):
    """Within the bound, and in all as near as the rounding of the result: fp32 sums add less than 1e-5 of it."""
    x = normals((M, K), M, t, dev)
    c, s, z = ops.quantize_int4_weight(normals((N, K), N, torch.float32, dev, K ** -0.5).to(t), group, zeros)
    ref = x.double() @ int4_weight(c, s, z, group, K).t()
    y = ops.linear_int4(x, c, s, z, group)
    assert_within(y, ref, int4_bound(x, s, z, group, t, ref), "y")
    least = (ref.to(t).double() - ref).norm()
    assert (y.double() - ref).norm() <= 1.1 * least + 1e-5 * ref.norm()


def test_strides_shapes_and_padding(dev):
    """Rows of x apart, on an odd address and with leading dimensions; words of codes apart; what stands behind K in the last words does not count."""
    K, N, t = 72, 40, torch.bfloat16
    x, q = ints((6, K), 3, 0, t, dev), torch.randint(0, 16, (N, K), generator=torch.Generator().manual_seed(1)).to(dev)
    s = torch.ones((N, 1), dtype=t, device=dev)
    c = pack_codes(q)
    want = (x.double() @ (q.double() - 8).t()).to(t)
    wide = torch.zeros((6, 99), dtype=t, device=dev)
    for at in (0, 3, 8):
        wide[:, at:at + K] = x
        assert torch.equal(ops.linear_int4(wide[:, at:at + K], c, s), want)
    assert torch.equal(ops.linear_int4(x.view(2, 3, K), c, s), want.view(2, 3, N))
    assert torch.equal(ops.linear_int4(x.t().contiguous().t(), c, s), want) and torch.equal(ops.linear_int4(x.repeat_interleave(2, 1)[:, ::2], c, s), want)
    part = c.clone()[:, :4 * -(-67 // 32)]
    assert torch.equal(ops.linear_int4(x[:, :67], part, s), (x[:, :67].double() @ (q[:, :67].double() - 8).t()).to(t))
    assert torch.equal(ops.linear_int4(x[0], c, s), want[0])
    assert torch.equal(ops.linear_int4(x[:1].expand(50, K), c, s), want[:1].expand(50, N))
    assert ops.linear_int4(x[:0], c, s).shape == (0, N)
    far = torch.zeros((N, 20), dtype=torch.int32, device=dev)
    far[:, 4:16] = c
    far[:, 4 + K // 8:] = -1
    assert torch.equal(ops.linear_int4(x, far[:, 4:16], s), want)
    assert torch.equal(ops.linear_int4(x.repeat(20, 1), far[:, 4:16], s.expand(N, 1)), want.repeat(20, 1))
    one = torch.ones((N, 3), dtype=t, device=dev)[:, :1].expand(N, 3)
    assert torch.equal(ops.linear_int4(x, c, one, group_size=32), want)


def test_rows_do_not_touch_each_other(dev):
    """An infinity or NaN stays in its row."""
    for M in (5, 40, 5000):
        x = normals((M, 256), M, torch.float16, dev)
        c, s, _ = ops.quantize_int4_weight(normals((48, 256), 1, torch.float16, dev))
        clean = ops.linear_int4(x, c, s)
        x[1, 3], x[3, 200] = float("inf"), float("nan")
        y = ops.linear_int4(x, c, s)
        assert bool(torch.isnan(y[[1, 3]]).all()) and torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])


def test_refusals(dev):
    x, w = normals((4, 64), 0, torch.bfloat16, dev), normals((16, 64), 1, torch.bfloat16, dev)
    c, s, _ = ops.quantize_int4_weight(w, 32)
    z = torch.zeros((16, 2), dtype=torch.uint8, device=dev)
    for bad in (lambda: ops.linear_int4(x, c, s, group_size=16), lambda: ops.linear_int4(x, c, s, group_size=64), lambda: ops.linear_int4(x[:, :31], c, s, group_size=32),
                lambda: ops.linear_int4(x, c[:, 1:], s, group_size=32), lambda: ops.linear_int4(x, c, s[:8], group_size=32), lambda: ops.linear_int4(x, c, s, z[:, :1], group_size=32),
                lambda: ops.linear_int4(x, c.t().contiguous().t(), s, group_size=32), lambda: ops.quantize_int4_weight(w, 100), lambda: ops.quantize_int4_weight(w[0]),
                lambda: ops.linear_int4(x[:, :0], c, s, group_size=32)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.linear_int4(x.float(), c, s, group_size=32), lambda: ops.linear_int4(x, c.long(), s, group_size=32), lambda: ops.linear_int4(x, c, s.half(), group_size=32),
                lambda: ops.linear_int4(x, c, s, z.int(), group_size=32), lambda: ops.quantize_int4_weight(w.double()), lambda: ops.linear_int4(x, c, s, group_size="32")):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.linear_int4(x.requires_grad_(), c, s, group_size=32), lambda: ops.quantize_int4_weight(w.requires_grad_(), 32)):
        with pytest.raises(RuntimeError, match="no gradients"):
            bad()
    with torch.no_grad():
        ops.linear_int4(x, c, s, group_size=32)


@pytest.mark.parametrize("M", [3, 100, 5000])
def test_captured_and_on_another_stream(dev, M):
    x = normals((M, 400), 0, torch.bfloat16, dev)
    c, s, z = ops.quantize_int4_weight(normals((136, 400), 1, torch.bfloat16, dev), 64, True)
    want = ops.linear_int4(x, c, s, z, 64)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.linear_int4(x, c, s, z, 64)
    stream.synchronize()
    assert torch.equal(got, want)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        a = ops.linear_int4(x, c, s, z, 64)
    with torch.cuda.graph(second, pool=first.pool()):
        b = ops.linear_int4(a[:, :136].repeat(1, 3)[:, :400], c, s, z, 64)
    for seed in (2, 3, 4):
        x.copy_(normals((M, 400), seed, torch.bfloat16, dev))
        first.replay(), second.replay()
        eager = ops.linear_int4(x, c, s, z, 64)
        torch.cuda.synchronize()
        assert torch.equal(a, eager) and torch.equal(b, ops.linear_int4(eager.repeat(1, 3)[:, :400], c, s, z, 64))
