"""ops.layernorm against the formulas in 64 bits: types, widths, strides, weights, gradients; bounds of dense_util.norm_bounds."""
import pytest
import torch

from dense_util import assert_within, norm_bounds, norm_reference, normals, rounding
from mortar_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _case(M, d, t, dev, seed, wt=None):
    x = normals((M, d), seed, torch.float32, dev) * (0.5 + torch.rand((M, 1), device=dev)) + normals((d,), seed + 1, torch.float32, dev, 0.5)
    wt = wt or t
    return x.to(t), (1 + normals((d,), seed + 2, torch.float32, dev, 0.1)).to(wt), normals((d,), seed + 3, wt, dev, 0.1), normals((M, d), seed + 4, t, dev)


def _check(x, w, b, dy, eps, got):
    want, bounds = norm_reference(x, w, b, eps, dy), norm_bounds(x, w, b, eps, dy)
    for name, g, r, e in zip(("y", "dx", "dw", "db"), got, want, bounds):
        if g is not None:
            assert_within(g, r, e if name in ("y", "dx") else e + rounding(g.dtype, r), name)


def _grads(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = ops.layernorm(*leaves, eps=eps)
    present = [t for t in leaves if t is not None]
    gr = iter(torch.autograd.grad(y, present, dy))
    return [y.detach()] + [next(gr) if t is not None else None for t in leaves]


# a row of one value; below, at and beyond a wave's vectors; odd; the widest held in registers; the loops behind them
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,d", [(1, 1), (1, 8), (3, 7), (5, 64), (4, 200), (9, 512), (2, 513), (7, 768), (6, 1023), (5, 2048), (3, 2056), (2, 8192), (3, 8191),
                                 (2, 16384), (2, 16392), (3, 9001)])
def test_values_and_gradients(dev, t, M, d):
    x, w, b, dy = _case(M, d, t, dev, 10 * d + M)
    _check(x, w, b, dy, 1e-5, _grads(x, w, b, dy))


# more rows than the workgroups take in one turn, and a number that no workgroup size divides
@pytest.mark.parametrize("M,d,t", [(2049, 96, torch.float32), (8195, 40, torch.bfloat16), (2500, 2048, torch.float16), (9001, 33, torch.float16), (1030, 4096, torch.bfloat16)])
def test_many_rows(dev, M, d, t):
    x, w, b, dy = _case(M, d, t, dev, 3 * M)
    _check(x, w, b, dy, 1e-5, _grads(x, w, b, dy))


@pytest.mark.parametrize("t", TYPES[:2], ids=str)
def test_fp32_weights_with_16_bit_rows(dev, t):
    for M, d in ((5, 768), (6, 35)):
        x, w, b, dy = _case(M, d, t, dev, 5, torch.float32)
        got = _grads(x, w, b, dy)
        assert got[0].dtype == got[1].dtype == t and got[2].dtype == got[3].dtype == torch.float32
        _check(x, w, b, dy, 1e-5, got)


def test_without_weight_or_bias(dev):
    x, w, b, dy = _case(6, 320, torch.bfloat16, dev, 77)
    for ww, bb in ((None, None), (w, None), (None, b)):
        _check(x, ww, bb, dy, 1e-3, _grads(x, ww, bb, dy, 1e-3))


def test_only_the_gradients_that_are_wanted(dev):
    x, w, b, dy = _case(70, 256, torch.float32, dev, 9)
    full = _grads(x, w, b, dy)
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        (g,) = torch.autograd.grad(ops.layernorm(*leaves), [leaves[i]], dy)
        assert torch.equal(g, full[i + 1])


def test_strides_and_offsets(dev):
    """Rows of a wider tensor, every other row, a transposed tensor, an odd address, one row repeated: the same bits as the copies."""
    base = normals((12, 520), 3, torch.bfloat16, dev)
    w, b = normals((200,), 4, torch.bfloat16, dev), normals((200,), 5, torch.bfloat16, dev)
    for x in (base[:, 8:208], base[:, 3:203], base[::2, 100:300], normals((200, 6), 6, torch.bfloat16, dev).t(), base[:1, :200].expand(5, 200),
              base[2:8, :400].reshape(6, 2, 200), base[0, 1:201]):
        ref = ops.layernorm(x.contiguous().clone(), w, b)
        assert_within(ops.layernorm(x, w, b).reshape(-1, 200), ref.double().reshape(-1, 200), 2 * rounding(torch.bfloat16, ref.double().reshape(-1, 200)), "strided")
        dy = normals(x.shape, 7, torch.bfloat16, dev)
        xl = x.detach().requires_grad_(True)
        (g,) = torch.autograd.grad(ops.layernorm(xl, w, b), [xl], dy)
        assert_within(g.reshape(-1, 200), norm_reference(x.reshape(-1, 200), w, b, 1e-5, dy.reshape(-1, 200))[1], norm_bounds(x.reshape(-1, 200), w, b, 1e-5, dy.reshape(-1, 200))[1], "strided dx")
    x = base[:, :200]
    xl = x.detach().requires_grad_(True)
    for dy in (normals((200, 12), 8, torch.bfloat16, dev).t(), torch.ones((), dtype=torch.bfloat16, device=dev).expand(12, 200)):
        (g,) = torch.autograd.grad(ops.layernorm(xl, w, b), [xl], dy)
        assert_within(g, norm_reference(x, w, b, 1e-5, dy)[1], norm_bounds(x, w, b, 1e-5, dy)[1], "dx of a strided dy")


def test_no_rows(dev):
    x = torch.empty((0, 64), dtype=torch.float32, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = ops.layernorm(x, w)
    gx, gw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
    assert y.shape == (0, 64) and gx.shape == (0, 64) and torch.equal(gw, torch.zeros(64, device=dev))


def test_rows_that_are_not_finite_stay_among_themselves(dev):
    x, w, b, dy = _case(9, 384, torch.bfloat16, dev, 21)
    good = _grads(x, w, b, dy)
    x2 = x.clone()
    x2[3, 5], x2[6, 0], x2[7, 383] = float("nan"), float("inf"), float("-inf")
    y, dx, dw, db = _grads(x2, w, b, dy)
    keep = [i for i in range(9) if i not in (3, 6, 7)]
    assert torch.equal(y[keep], good[0][keep]) and torch.equal(dx[keep], good[1][keep]) and torch.equal(db, good[3])
    assert bool(y[[3, 6, 7]].isnan().all()) and bool(dx[[3, 6, 7]].isnan().all())


def test_constant_rows_and_large_means(dev):
    """A row of one value is all bias; values far from zero keep their variance (it is formed from centred values)."""
    w, b = normals((256,), 1, torch.float32, dev), normals((256,), 2, torch.float32, dev)
    assert torch.equal(ops.layernorm(torch.full((3, 256), 1.5, device=dev), w, b), b.expand(3, 256))
    x = 4096 + normals((4, 256), 3, torch.float32, dev)
    assert_within(ops.layernorm(x, w, b), norm_reference(x, w, b, 1e-5), norm_bounds(x, w, b, 1e-5), "large mean")


def test_gradient_against_differences(dev):
    """Along a direction v: (L(x + e v) - L(x - e v)) / 2e with L = <dy, y>, evaluated in 64 bits on the fp32 results.  The difference
    quotient is off by e^2 / 6 times a third derivative of order one per value (1e-4 of sum |dy v|), the results by 1e-6 / e."""
    x, w, b, dy = _case(6, 160, torch.float32, dev, 31)
    _, dx, dw, db = _grads(x, w, b, dy)
    for i, (t, grad) in enumerate(((x, dx), (w, dw), (b, db))):
        v, e = normals(t.shape, 40 + i, torch.float32, dev), 2.0 ** -6
        at = lambda s: float((dy.double() * ops.layernorm(*[p + s * v if j == i else p for j, p in enumerate((x, w, b))]).double()).sum())
        want = float((grad.double() * v.double()).sum())
        scale = float((dy.abs().double()).sum() * v.abs().max())
        assert abs((at(e) - at(-e)) / (2 * e) - want) <= (e * e / 6 * 8 + 2e-6 / e) * scale


def test_same_bits_every_time_and_on_another_stream(dev):
    x, w, b, dy = _case(5000, 768, torch.bfloat16, dev, 51)
    first = _grads(x, w, b, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = _grads(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(s)
    for a, c in zip(first, other):
        assert torch.equal(a, c)


def test_replayed_from_a_graph(dev):
    x, w, b, dy = _case(300, 768, torch.bfloat16, dev, 61)
    xs, dys = x.clone(), dy.clone()
    leaves = [xs.requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]

    def step():
        y = ops.layernorm(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dys))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        nx, ndy = normals(x.shape, 70 + i, torch.bfloat16, dev), normals(x.shape, 80 + i, torch.bfloat16, dev)
        with torch.no_grad():
            xs.copy_(nx), dys.copy_(ndy)
        g.replay()
        want = _grads(nx, w, b, ndy)
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)


def test_refusals(dev):
    x = torch.zeros((4, 32), device=dev)
    w = torch.ones(32, device=dev)
    with pytest.raises(TypeError):
        ops.layernorm(x.double())
    with pytest.raises(TypeError):
        ops.layernorm(x, w.half())
    with pytest.raises(TypeError):
        ops.layernorm(x.half(), w.half(), w)
    with pytest.raises(ValueError):
        ops.layernorm(x, w[:31])
    with pytest.raises(ValueError):
        ops.layernorm(x, w, w.view(1, 32))
    with pytest.raises(ValueError):
        ops.layernorm(torch.zeros((), device=dev))
    with pytest.raises(ValueError):
        ops.layernorm(x, w, eps=-1.0)
    with pytest.raises(TypeError):
        ops.layernorm([1.0])
    with pytest.raises(RuntimeError):
        ops.layernorm(x, w.cpu())
    xl = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.layernorm(xl, w).sum(), [xl])
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(ops.layernorm(xl, w).sum(), [xl], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda r: ops.layernorm(r, w))(x)
